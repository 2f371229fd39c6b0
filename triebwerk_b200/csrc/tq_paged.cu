// extern "C" calls over paged packed caches (declared in include/triebwerk_b200.h): a translation unit of its own, so that it compiles
// beside tq_capi.cu.

#include <atomic>

#include "tq_host.cuh"
#include "tq_paged.cuh"
#include "tq_paged_prefill.cuh"
#include "tq_paged_rows.cuh"

using namespace tq;

static inline cudaStream_t cs(tq_stream_t s) { return reinterpret_cast<cudaStream_t>(s); }

static inline bool use_pdl() {
    static const bool on = !(getenv("TQ_PDL") && atoi(getenv("TQ_PDL")) == 0);
    return on;
}

// The status word of all paged calls on a device: a wait that gave up, a shared-memory layout refused.
static __device__ int g_paged_status;
static int paged_status_word(int** out) {
    constexpr int KNOWN = 64;
    static std::atomic<int*> known[KNOWN];
    int dev = 0;
    TQ_CUDA(cudaGetDevice(&dev));
    if (dev < KNOWN && (*out = known[dev].load(std::memory_order_acquire))) return TQ_OK;
    void* a = nullptr;
    TQ_CUDA(cudaGetSymbolAddress(&a, g_paged_status));
    *out = (int*)a;
    if (dev < KNOWN) known[dev].store(*out, std::memory_order_release);
    return TQ_OK;
}

static bool page_size_ok(int page_size) { return page_size >= TILE_TOKENS && page_size <= 65536 && (page_size & (page_size - 1)) == 0; }
static int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}
static int check_pages(int table_stride, int table_width, int num_pages, int page_size) {
    if (!page_size_ok(page_size)) return TQ_ERR_UNSUPPORTED;
    if (num_pages <= 0 || table_width <= 0 || table_stride < table_width) return TQ_ERR_ARG;
    if ((long long)num_pages * page_size >= (1ll << 31) || (long long)table_width * page_size >= (1ll << 31)) return TQ_ERR_UNSUPPORTED;
    return TQ_OK;
}
// Cache arrays and R are moved 16 bytes at a time, norms and rows of fewer bytes by their own size.
static bool aligned(std::initializer_list<const void*> p, unsigned to) {
    uintptr_t all = 0;
    for (const void* a : p) all |= (uintptr_t)a;
    return (all & (to - 1u)) == 0;
}
// An array: `rows` rows of `width` bytes, `stride` apart (one row: any).
struct Span {
    const void* at;
    long long width, stride, rows;
};
// Do two arrays share memory?  Rows of either may lie between the other's (columns of one wider array).
static bool overlap(const Span& a, const Span& b) {
    if (a.rows <= 0 || a.width <= 0 || b.rows <= 0 || b.width <= 0) return false;
    const long long d = (long long)((uintptr_t)b.at - (uintptr_t)a.at);  // row j of b begins at d + j * b.stride, row i of a at i * a.stride
    const long long a_last = (a.rows - 1) * a.stride, b_last = d + (b.rows - 1) * b.stride;
    if (a_last + a.width <= d || b_last + b.width <= 0) return false;
    if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) {  // (that of one wider array: no loop)
        const long long r = (d % a.stride + a.stride) % a.stride;
        return r < a.width || r > a.stride - b.width;
    }
    // the first row of either that ends behind the other's row, in turn
    auto past = [](long long begin, const Span& s, long long first) { return begin + s.width <= first ? (first - begin - s.width) / s.stride + 1 : 0; };
    for (long long i = 0, j = 0;;) {
        const long long skip_a = past(i * a.stride, a, d + j * b.stride);
        if ((i += skip_a) >= a.rows) return false;
        const long long skip_b = past(d + j * b.stride, b, i * a.stride);
        if ((j += skip_b) >= b.rows) return false;
        if (skip_b == 0) return true;  // (row i of a ends behind row j's begin, row j of b behind row i's)
    }
}
static Span half_rows(const void* at, long long rows, long long width, long long stride) { return {at, 2 * width, 2 * stride, rows}; }
static Span block(const void* at, long long bytes) { return {at, bytes, bytes, at ? 1 : 0}; }
// Does anything that a call writes share memory with something else that it writes, or with something that it reads?
static bool clash(std::initializer_list<Span> written, std::initializer_list<Span> read) {
    for (const Span* w = written.begin(); w != written.end(); ++w) {
        for (const Span* o = written.begin(); o != w; ++o)
            if (overlap(*w, *o)) return true;
        for (const Span& r : read)
            if (overlap(*w, r)) return true;
    }
    return false;
}
constexpr long long ROTATION_BYTES = 2ll * HEAD_DIM * HEAD_DIM;

extern "C" {

int tq_paged_status(tq_stream_t s) {
    int* word = nullptr;
    int r = paged_status_word(&word);
    return r != TQ_OK ? r : tq_workspace_status(word, s);
}

int tq_page_plan(int* block_table, int table_stride, int table_width, int* free_pages, const int* free_count, int* free_count_out, int num_pages,
                 int page_size, const int* context_lens, const int* new_tokens, const unsigned char* finished, int G, int* seq_lens,
                 int* query_start, long long* slots, int* positions, int T, tq_stream_t s) {
    int r = check_pages(table_stride, table_width, num_pages, page_size);
    if (r != TQ_OK) return r;
    if (!block_table || !free_pages || !free_count || !free_count_out || !context_lens || !new_tokens || !seq_lens || !query_start || G <= 0 || T < 0 || (T > 0 && !slots))
        return TQ_ERR_ARG;
    if (!aligned({block_table, free_pages, free_count, free_count_out, context_lens, new_tokens, seq_lens, query_start, positions}, 4) || !aligned({slots}, 8)) return TQ_ERR_ARG;
    if (clash({Span{block_table, 4ll * table_width, 4ll * table_stride, G}, block(free_pages, 4ll * num_pages), block(free_count_out, 4), block(seq_lens, 4ll * G),
               block(query_start, 4ll * G + 4), block(slots, 8ll * T), block(positions, 4ll * T)},
              {block(free_count == free_count_out ? nullptr : free_count, 4), block(context_lens == seq_lens ? nullptr : context_lens, 4ll * G), block(new_tokens, 4ll * G),
               block(finished, G)}))
        return TQ_ERR_ARG;
    PagePlanParams p{};
    p.table = block_table; p.free_pages = free_pages; p.free_count = free_count; p.free_count_out = free_count_out;
    p.context = context_lens; p.new_tokens = new_tokens; p.finished = finished; p.lens = seq_lens; p.start = query_start; p.slots = slots; p.positions = positions;
    p.G = G; p.T = T; p.num_pages = num_pages; p.table_stride = table_stride; p.width = table_width; p.page_shift = log2_of(page_size);
    r = launch_kernel(page_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, cs(s), use_pdl(), p);
    if (r != TQ_OK || T <= PLAN_ONE_LAUNCH) return r;
    const int ctas = std::min((T + SLOTS_THREADS - 1) / SLOTS_THREADS, 4 * device_props().sm_count);
    return launch_kernel(page_slots_kernel, dim3((unsigned)ctas), dim3(SLOTS_THREADS), 0, cs(s), use_pdl(), p);
}

// (head_dim, head counts, bits, rows)
static int check_rows(int T, int Hkv, int head_dim, long long kv_stride, int bits, long long total_rows) {
    if (head_dim != HEAD_DIM) return TQ_ERR_UNSUPPORTED;
    if (T < 0 || Hkv <= 0 || (bits != 2 && bits != 4) || total_rows <= 0 || kv_stride < (long long)Hkv * HEAD_DIM || kv_stride % 8 != 0) return TQ_ERR_ARG;
    if (total_rows >= (1ll << 31) || (long long)T * Hkv >= (1ll << 30) || kv_stride >= (1ll << 30)) return TQ_ERR_UNSUPPORTED;
    return TQ_OK;
}

int tq_paged_append(uint8_t* ck_q, void* k_norms, uint8_t* cv_q, void* v_norms, const void* k_buf, const void* v_buf, const void* rotation,
                    const long long* slots, long long total_rows, int T, int num_kv_heads, int head_dim, long long kv_stride, int bits, tq_stream_t s) {
    int r = check_rows(T, num_kv_heads, head_dim, kv_stride, bits, total_rows);
    if (r != TQ_OK) return r;
    if (!ck_q || !k_norms || !cv_q || !v_norms || !rotation || (T > 0 && (!k_buf || !v_buf || !slots))) return TQ_ERR_ARG;
    if (!aligned({ck_q, cv_q, k_buf, v_buf, rotation}, 16) || !aligned({k_norms, v_norms}, 2) || !aligned({slots}, 8)) return TQ_ERR_ARG;
    if (T == 0) return TQ_OK;
    const long long codes = total_rows * num_kv_heads * (HEAD_DIM * bits / 8), norms = 2 * total_rows * num_kv_heads;
    if (clash({block(ck_q, codes), block(cv_q, codes), block(k_norms, norms), block(v_norms, norms)},
              {half_rows(k_buf, T, num_kv_heads * HEAD_DIM, kv_stride), half_rows(v_buf, T, num_kv_heads * HEAD_DIM, kv_stride), block(rotation, ROTATION_BYTES), block(slots, 8ll * T)}))
        return TQ_ERR_ARG;
    int* status = nullptr;
    r = paged_status_word(&status);
    if (r != TQ_OK) return r;
    // A CTA per token (2 * KV heads <= 16 vectors) while those are one turn of two per SM, tiles of 128 vectors behind that.  (us for 64, 148, 296, 444,
    // 592 tokens, token / tile: 4-bit 8 KV heads 5.1 / 6.6, 5.6 / 6.6, 6.8 / 7.4, 10.4 / 7.5, 11.0 / 7.6; 2-bit 4 KV heads 4.5 / 6.5, 4.6 / 6.5, 5.5 / 6.4, 8.3 /
    // 6.5, 8.5 / 6.5.)
    if (num_kv_heads <= 8 && T <= 2 * device_props().sm_count) {
        LayerPrepParams p{};
        p.ck = ck_q; p.cv = cv_q; p.kn = (__half*)k_norms; p.vn = (__half*)v_norms;
        p.new_k = (const __half*)k_buf; p.new_v = (const __half*)v_buf; p.rotation = (const __half*)rotation; p.rot_copies = 1; p.status = status;
        p.G = T; p.H = 0; p.Hkv = num_kv_heads;
        p.slots = slots; p.total_rows = total_rows; p.kv_stride = kv_stride;
        const dim3 grid((unsigned)std::min(T, 2 * device_props().sm_count));
        return bits == 4 ? launch_kernel(layer_prep_kernel<4, true>, grid, dim3(PREP_THREADS), 0, cs(s), use_pdl(), p)
                         : launch_kernel(layer_prep_kernel<2, true>, grid, dim3(PREP_THREADS), 0, cs(s), use_pdl(), p);
    }
    PrefillTcParams t{};
    t.ck = ck_q; t.cv = cv_q; t.kn = (__half*)k_norms; t.vn = (__half*)v_norms;
    t.k_buf = (const __half*)k_buf; t.v_buf = (const __half*)v_buf; t.rotation = (const __half*)rotation; t.status = status;
    t.row_base = slots; t.total_rows = total_rows;
    t.n_seq = T; t.T = 1; t.Hkv = num_kv_heads; t.kv_dim = (int)kv_stride; t.bits = bits;
    const long long tiles = 2 * (((long long)T * num_kv_heads + TC_TILE - 1) / TC_TILE);
    CUtensorMap tmk{}, tmv{};
    const bool tma = make_append_input_map(&tmk, k_buf, T, num_kv_heads, t.kv_dim) == TQ_OK && make_append_input_map(&tmv, v_buf, T, num_kv_heads, t.kv_dim) == TQ_OK;
    auto kernel = tma ? prefill_append_tc_kernel<false, true, false, true> : prefill_append_tc_kernel<false, false, false, true>;
    r = ensure_dynamic_smem((const void*)kernel, TC_DYN_SMEM);
    if (r != TQ_OK) return r;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)std::min<long long>(tiles, (long long)TC_CTAS_PER_SM * device_props().sm_count));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = TC_DYN_SMEM;
    cfg.stream = cs(s);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl() ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, tmk, tmv, t));
}

int tq_paged_read(void* k_out, void* v_out, const uint8_t* ck_q, const void* k_norms, const uint8_t* cv_q, const void* v_norms, const void* rotation,
                  const long long* slots, long long total_rows, int T, int num_kv_heads, int head_dim, long long kv_stride, int bits, tq_stream_t s) {
    int r = check_rows(T, num_kv_heads, head_dim, kv_stride, bits, total_rows);
    if (r != TQ_OK) return r;
    if (!ck_q || !k_norms || !cv_q || !v_norms || !rotation || (T > 0 && (!k_out || !v_out || !slots))) return TQ_ERR_ARG;
    if (!aligned({ck_q, cv_q, rotation, k_out, v_out}, 16) || !aligned({k_norms, v_norms}, 2) || !aligned({slots}, 8)) return TQ_ERR_ARG;
    if (T == 0) return TQ_OK;
    const long long codes = total_rows * num_kv_heads * (HEAD_DIM * bits / 8), norms = 2 * total_rows * num_kv_heads;
    if (clash({half_rows(k_out, T, num_kv_heads * HEAD_DIM, kv_stride), half_rows(v_out, T, num_kv_heads * HEAD_DIM, kv_stride)},
              {block(ck_q, codes), block(cv_q, codes), block(k_norms, norms), block(v_norms, norms), block(rotation, ROTATION_BYTES), block(slots, 8ll * T)}))
        return TQ_ERR_ARG;
    PagedReadParams p{};
    p.ck = ck_q; p.kn = (const __half*)k_norms; p.cv = cv_q; p.vn = (const __half*)v_norms; p.rotation = (const __half*)rotation;
    p.slots = slots; p.k_out = (__half*)k_out; p.v_out = (__half*)v_out; p.total_rows = total_rows; p.stride = kv_stride; p.T = T; p.Hkv = num_kv_heads;
    const long long tiles = 2 * (((long long)T * num_kv_heads + READ_VECTORS - 1) / READ_VECTORS);
    const dim3 grid((unsigned)std::min<long long>(tiles, 2ll * device_props().sm_count));
    return bits == 4 ? launch_kernel(paged_read_kernel<4>, grid, dim3(READ_THREADS), 0, cs(s), use_pdl(), p)
                     : launch_kernel(paged_read_kernel<2>, grid, dim3(READ_THREADS), 0, cs(s), use_pdl(), p);
}

}  // extern "C"

// How a prefill call's work is cut.  The host knows the tokens of all requests together, so it goes by their mean.
struct PrefillCut {
    bool small, large;   // whether there may be requests of up to, of more than ROWS_MOST score rows
    int ncb, parts;      // small ones: row blocks of 8 per CTA, parts of a request's tokens
    int mt, most_parts;  // large ones: blocks of 128 rows per CTA; parts that a block's tiles may be cut into, 1: not cut
    bool mostly_small;   // requests are small in the mean: none may be large, or one
};
constexpr int SPLIT_SMS = 160, MAX_SPLITS = 16;
// Rows of partial sums that those calls may write.  Large requests are cut only while parts * blocks of 128 rows <= the SMs and the parts fit; small ones, of which a request
// has 32 rows per KV head at most, into as many parts as fit.
static size_t large_rows(long long T, long long H) { return (size_t)std::min<long long>(MAX_SPLITS * T * H, (long long)SPLIT_SMS * PFT_ROWS); }
static size_t small_rows(long long T, long long G, long long H) {
    return (size_t)std::max(std::min(T, (long long)ROWS_MOST * G) * H, std::min<long long>(MAX_SPLITS * T * H, 8ll * SPLIT_SMS * ROWS_MOST));
}
static PrefillCut prefill_cut(int T, int G, int H, int Hkv, int most) {
    const long long sms = std::min(device_props().sm_count, SPLIT_SMS), grp = H / Hkv, qt = PFT_ROWS / grp, mean = (T + G - 1) / G;
    PrefillCut c{};
    c.small = grp <= ROWS_MOST && (G > 1 || T * grp <= ROWS_MOST);
    c.large = grp > ROWS_MOST || T * grp > ROWS_MOST;
    // Small ones.  A CTA takes start + turn * (its warps' turns of 16 tokens), us by row blocks per CTA below; as many at a time as the SMs hold, and part of
    // a turn more where there are several (contexts differ; less of it where the longest come first).  Up to 16 rows in one CTA; 17 to 24, where all requests
    // have as many (T is a multiple of G), in one of three blocks, alone on its SM, or in two of two.  Requests that differ count for half as many rows again as
    // their mean.  (Two / three blocks, best parts of each, us: 32/8 heads 32 x 5 behind 4000 2-bit 137 / 115, 4-bit 157 / 140; 4-bit 8 x 5 behind 4000 51 / 47,
    // 64 x 6 behind 1000 112 / 125; 2-bit 2 x 5 behind 30000 74 / 59; 32/4 16 x 3 behind 6000 68 / 59; 2-bit 32/8 32 x 1 to 5 behind 2000 to 4000 86 / 96.  By
    // parts 1, 2, 3, 4: the last, two blocks 87 / 86 / 92 / 103; 4-bit 8 x 5, three blocks 69 / 47 / 61 / 58; 16/8 64 x 1 behind 2000 75 / 85 / 97 / 104, 48 x 1
    // behind 100 to 4000 60 / 69 / 83 / 95; 32/8 32 x 5 behind 1000 to 8000 146 / 170 / 197 / 209.)
    const bool alike = T % G == 0;
    const long long rows = std::min(mean * grp, (long long)ROWS_MOST), tiles = (most + 15) / 16;
    const long long most_parts = std::min<long long>(MAX_SPLITS, (long long)small_rows(T, G, H) / std::max(1ll, std::min<long long>(T, G * (ROWS_MOST / grp)) * H));
    double best = 1e30;
    for (int ncb = rows <= 8 ? 1 : 2; ncb <= (rows <= 8 ? 1 : alike && rows > 16 && rows <= 24 ? 3 : 2); ++ncb) {
        const double start = ncb == 1 ? 5.0 : ncb == 2 ? 7.0 : 11.0, turn = ncb == 1 ? 1.6 : ncb == 2 ? 2.4 : 2.7;
        const long long warps = ncb == 3 ? ROWS_WARPS<3> : ROWS_WARPS<2>, room = ncb == 3 ? sms : 2 * sms;
        const long long ctas = Hkv * std::min<long long>(G, T) * (((alike ? rows : std::min(rows * 3 / 2, (long long)ROWS_MOST)) + 8 * ncb - 1) / (8 * ncb));
        for (long long parts = 1; parts <= std::max(1ll, most_parts); ++parts) {
            const double turns = ctas * parts <= room ? 1.0 : (G <= ROWS_SORTED ? 0.25 : 0.5) + (double)(ctas * parts) / (double)room;
            const double us = turns * (start + turn * ((tiles + warps * parts - 1) / (warps * parts)));
            if (us < best) {
                best = us;
                c.ncb = ncb;
                c.parts = (int)parts;
            }
        }
    }
    // Two blocks a CTA take 1.3 to 1.4 times as long as one, and the SMs serve a turn of CTAs at a time.  (us, one / two: 4-bit 32/8 heads 1 x 512 tokens
    // 16.6 / 21.3, 1 x 2048 91.6 / 62.0, 4 x 512 52.4 / 39.6, 1 x 1024 behind 8192 273 / 209; 2-bit 16/8 2 x 512 behind 8192 139 / 186, 4 x 512
    // 30.7 / 24.6, 4 x 2048 behind 4096 583 / 437.)
    const long long blocks1 = Hkv * G * ((mean + qt - 1) / qt), blocks2 = Hkv * G * ((mean + 2 * qt - 1) / (2 * qt));
    c.mt = mean > qt && 27 * ((blocks2 + sms - 1) / sms) < 20 * ((blocks1 + sms - 1) / sms) ? 2 : 1;
    // Blocks that leave half of the SMs idle are cut (2-bit 16/8 1 x 256 behind 20000: 294 uncut, 99).  Where requests are small in the mean or differ, they may: all tokens
    // but a few may be one request's, beside single tokens that have no block, so the fewest blocks that T can make decide, and the kernel counts what there is.
    // (Never cut / so, 4-bit 32/8 heads: 63 single tokens beside 64 behind 30000 560 / 186, 15 beside 200 behind 16000 297 / 185, 12 x 3 to 20 behind 4000 107 / 81,
    // 31 x 1 and 64 behind 8000 181 / 87; no block to cut in 32 x 1 to 5 behind 2000 to 4000 86.7 / 87.2, too many in 16 x 9 to 20 behind 4000 77.5 / 82.2.)
    c.mostly_small = mean * grp <= ROWS_MOST;
    const long long fewest = alike && !c.mostly_small ? blocks1 : std::min(blocks1, Hkv * ((T + qt - 1) / qt));
    c.most_parts = c.mt == 2 || 2 * fewest > sms ? 1 : (int)std::max(1ll, std::min({(long long)most / (4 * PFT_KT), (long long)MAX_SPLITS, (long long)large_rows(T, H) / ((long long)T * H)}));
    return c;
}
extern "C" {

size_t tq_paged_workspace_bytes(int T, int G, int num_heads) {
    if (T < 0 || G <= 0 || num_heads <= 0) return 0;
    return std::max(carve_full(nullptr, G, num_heads).bytes, (large_rows(T, num_heads) + small_rows(T, G, num_heads)) * PART_STRIDE * sizeof(float));
}

// What both attentions check of their arguments.
static int check_attention(const void* out, const void* q, const uint8_t* ck, const uint8_t* cv, const void* kn, const void* vn, const void* rotation,
                           const int* table, int table_stride, int table_width, const int* lens, int num_pages, int page_size, int T, int G, int H, int Hkv,
                           int head_dim, int q_stride, int out_stride, int bits) {
    int r = check_pages(table_stride, table_width, num_pages, page_size);
    if (r != TQ_OK) return r;
    if (head_dim != HEAD_DIM) return TQ_ERR_UNSUPPORTED;
    if (G <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || (bits != 2 && bits != 4)) return TQ_ERR_ARG;
    if ((long long)q_stride < (long long)H * HEAD_DIM || (long long)out_stride < (long long)H * HEAD_DIM || q_stride % 8 != 0 || out_stride % 8 != 0) return TQ_ERR_ARG;
    if (!ck || !cv || !kn || !vn || !rotation || !table || !lens || (T > 0 && (!out || !q))) return TQ_ERR_ARG;
    if (!aligned({out, q, ck, cv, kn, vn, rotation}, 16) || !aligned({table, lens}, 4)) return TQ_ERR_ARG;
    return TQ_OK;
}
// ... and what they write: results and workspace (T query rows; `start` of prefill alone).
static bool attention_clash(const void* out, const void* q, const uint8_t* ck, const uint8_t* cv, const void* kn, const void* vn, const void* rotation, const int* table,
                            int table_stride, int table_width, const int* lens, const int* start, long long rows, int T, int G, int H, int Hkv, int q_stride, int out_stride,
                            int bits, const void* workspace) {
    const long long codes = rows * Hkv * (HEAD_DIM * bits / 8), norms = 2 * rows * Hkv;
    return clash({half_rows(out, T, H * HEAD_DIM, out_stride), block(workspace, (long long)tq_paged_workspace_bytes(T, G, H))},
                 {half_rows(q, T, H * HEAD_DIM, q_stride), block(ck, codes), block(cv, codes), block(kn, norms), block(vn, norms), block(rotation, ROTATION_BYTES),
                  Span{table, 4ll * table_width, 4ll * table_stride, G}, block(lens, 4ll * G), block(start, 4ll * G + 4)});
}

int tq_paged_decode_attention(void* out, const void* q, const uint8_t* ck_q, const uint8_t* cv_q, const void* k_norms, const void* v_norms,
                              const void* rotation, const int* block_table, int table_stride, int table_width, const int* seq_lens, int num_pages,
                              int page_size, int G, int num_heads, int num_kv_heads, int head_dim, int q_stride, int out_stride, int bits,
                              void* workspace, size_t workspace_bytes, tq_stream_t s) {
    int r = check_attention(out, q, ck_q, cv_q, k_norms, v_norms, rotation, block_table, table_stride, table_width, seq_lens, num_pages, page_size, G, G,
                            num_heads, num_kv_heads, head_dim, q_stride, out_stride, bits);
    if (r != TQ_OK) return r;
    if (!workspace || workspace_bytes < tq_paged_workspace_bytes(G, G, num_heads) || !aligned({workspace}, 256)) return TQ_ERR_WORKSPACE;
    const int H = num_heads, Hkv = num_kv_heads, most = table_width * page_size, head_blocks = (H / Hkv + CD_HEADS - 1) / CD_HEADS;
    if (G > 65535 || (long long)Hkv * head_blocks > 65535) return TQ_ERR_UNSUPPORTED;
    const long long rows = (long long)num_pages * page_size;
    if (attention_clash(out, q, ck_q, cv_q, k_norms, v_norms, rotation, block_table, table_stride, table_width, seq_lens, nullptr, rows, G, G, H, Hkv, q_stride, out_stride, bits,
                        workspace))
        return TQ_ERR_ARG;
    int* status = nullptr;
    r = paged_status_word(&status);
    if (r != TQ_OK) return r;
    // The streaming form numbers the tiles of all requests with 32 bits.  Rows of the table may name the same pages, so the cache's size does not bound them:
    // below 2^28 the sums stay clear of overflow, and of the distance that stands for no prefetch.
    constexpr int MOST_TILES = 1 << 28;
    const bool streams = fast_shape(H, Hkv, true) && G <= FUSED_MAX_G && (long long)G * ((most + TILE_TOKENS - 1) / TILE_TOKENS) < MOST_TILES;
    if (!streams || cluster_layer_faster(bits, G, Hkv, H / Hkv, (long long)G * most, most, LayerCaller::Paged)) {
        ClusterDecodeParams p{};
        p.ck = ck_q; p.cv = cv_q; p.kn = (const __half*)k_norms; p.vn = (const __half*)v_norms; p.q = (const __half*)q; p.rotation = (const __half*)rotation;
        p.out = (__half*)out; p.positions = seq_lens; p.capacity_rows = most; p.max_seq_len = most; p.status = status;
        p.G = G; p.H = H; p.Hkv = Hkv; p.q_dim = q_stride; p.out_dim = out_stride; p.head_blocks = head_blocks;
        p.block_table = block_table; p.table_stride = table_stride; p.page_shift = log2_of(page_size); p.num_pages = num_pages;
        return launch_cluster_decode<false, true>(bits, p, 1, 1, most, cs(s), use_pdl());
    }
    const FullWorkspace fw = carve_full(workspace, G, H);
    CUtensorMap tmK, tmV;
    r = make_code_map(&tmK, ck_q, rows, Hkv * (bits == 4 ? 64 : 32));
    if (r == TQ_OK) r = make_code_map(&tmV, cv_q, rows, Hkv * (bits == 4 ? 64 : 32));
    if (r != TQ_OK) return r;
    LayerPrepParams lp{};
    lp.q = (const __half*)q; lp.rotation = (const __half*)rotation; lp.rot_copies = 1; lp.rotation_t = fw.rot_t; lp.status = status;
    if (bits == 2 && Hkv == 8) lp.q_rot32 = fw.w.q_rot;
    else lp.q_rot16 = (__half*)fw.w.q_rot;
    lp.G = G; lp.H = H; lp.Hkv = Hkv; lp.q_dim = q_stride;
    r = launch_layer_prep(bits, lp, cs(s), use_pdl());
    if (r != TQ_OK) return r;
    AttnParams p{};
    p.ck = ck_q; p.cv = cv_q; p.kn = (const __half*)k_norms; p.vn = (const __half*)v_norms;
    p.q_rot16 = lp.q_rot16; p.q_rot32 = lp.q_rot32; p.rotation_t = fw.rot_t; p.out = (__half*)out;
    p.positions = seq_lens; p.partials = fw.w.partials; p.status = status; p.total_rows = rows;
    p.G = G; p.H = H; p.Hkv = Hkv; p.q_dim = out_stride; p.n_layers = 1; p.l2_ahead = MOST_TILES;
    p.block_table = block_table; p.table_stride = table_stride; p.page_shift = log2_of(page_size); p.num_pages = num_pages; p.most_tokens = most;
    const int ctas = attention_ctas(G, most);
    if (Hkv == 8) r = bits == 4 ? launch_attention_t<4, 8, 1, true>(tmK, tmV, p, ctas, cs(s), use_pdl()) : launch_attention_t<2, 8, 1, true>(tmK, tmV, p, ctas, cs(s), use_pdl());
    else r = bits == 4 ? launch_attention_t<4, 4, 1, true>(tmK, tmV, p, ctas, cs(s), use_pdl()) : launch_attention_t<2, 4, 1, true>(tmK, tmV, p, ctas, cs(s), use_pdl());
    if (r != TQ_OK) return r;
    MergeLayerParams m{};
    m.partials = p.partials; m.positions = seq_lens; m.rotation_t = fw.rot_t; m.out = (__half*)out; m.G = G; m.H = H; m.q_dim = out_stride;
    m.workers = ctas * ATTN_GROUPS; m.most_tokens = most;
    return launch_merge_layer<true>(m, cs(s), use_pdl());
}

}  // extern "C"

template <int BITS, int MT, bool SPLIT>
static int launch_paged_prefill(const CUtensorMap& tmQ, const CUtensorMap& tmR, const PagedPrefillParams& p, dim3 grid, cudaStream_t s) {
    auto kernel = paged_prefill_kernel<BITS, MT, SPLIT>;
    int r = ensure_dynamic_smem((const void*)kernel, PpfSmem::BYTES);
    if (r != TQ_OK) return r;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(PPF_THREADS);
    cfg.dynamicSmemBytes = PpfSmem::BYTES;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl() ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, tmQ, tmR, p));
}

template <int BITS, int NCB>
static int launch_rows(const PagedRowsParams& p, dim3 grid, cudaStream_t s) {
    constexpr size_t smem = rows_smem_bytes<BITS>();
    const int r = ensure_dynamic_smem((const void*)paged_rows_kernel<BITS, NCB>, smem);
    return r != TQ_OK ? r : launch_kernel(paged_rows_kernel<BITS, NCB>, grid, dim3(ROWS_THREADS<NCB>), smem, s, use_pdl(), p);
}

extern "C" {

int tq_paged_prefill_attention(void* out, const void* q, const uint8_t* ck_q, const uint8_t* cv_q, const void* k_norms, const void* v_norms,
                               const void* rotation, const int* block_table, int table_stride, int table_width, const int* seq_lens,
                               const int* query_start, int num_pages, int page_size, int T, int G, int num_heads, int num_kv_heads, int head_dim,
                               int q_stride, int out_stride, int bits, void* workspace, size_t workspace_bytes, tq_stream_t s) {
    int r = check_attention(out, q, ck_q, cv_q, k_norms, v_norms, rotation, block_table, table_stride, table_width, seq_lens, num_pages, page_size, T, G,
                            num_heads, num_kv_heads, head_dim, q_stride, out_stride, bits);
    if (r != TQ_OK) return r;
    if (T < 0 || !query_start || !aligned({query_start}, 4)) return TQ_ERR_ARG;
    const int H = num_heads, Hkv = num_kv_heads, grp = H / Hkv, most = table_width * page_size;
    if (!prefill_attn_shape(H, Hkv)) return TQ_ERR_UNSUPPORTED;
    if (!workspace || workspace_bytes < tq_paged_workspace_bytes(T, G, H) || !aligned({workspace}, 256)) return TQ_ERR_WORKSPACE;
    if (T == 0) return TQ_OK;
    if ((long long)T * H >= (1ll << 31) || G > 65535) return TQ_ERR_UNSUPPORTED;
    if (attention_clash(out, q, ck_q, cv_q, k_norms, v_norms, rotation, block_table, table_stride, table_width, seq_lens, query_start, (long long)num_pages * page_size, T, G, H,
                        Hkv, q_stride, out_stride, bits, workspace))
        return TQ_ERR_ARG;
    int* status = nullptr;
    r = paged_status_word(&status);
    if (r != TQ_OK) return r;
    const PrefillCut cut = prefill_cut(T, G, H, Hkv, most);
    const int shift = log2_of(page_size), most_small = ROWS_MOST / grp;  // new tokens of a small request
    float* const small_sums = (float*)workspace + large_rows(T, H) * PART_STRIDE;
    PagedMergeParams m{};
    m.partials = (const float*)workspace; m.small_partials = small_sums; m.rotation = (const __half*)rotation; m.start = query_start; m.out = (__half*)out;
    m.T = T; m.G = G; m.H = H; m.Hkv = Hkv; m.grp = grp; m.out_stride = out_stride; m.small_rows = cut.small ? ROWS_MOST : 0;
    if (cut.large) {
        const int qt = PFT_ROWS / grp, bt = cut.mt * qt;
        const long long requests = std::min<long long>(G, cut.small ? T / (most_small + 1) : T), ctas = (long long)Hkv * (T / bt + requests);
        if (ctas >= (1ll << 31)) return TQ_ERR_UNSUPPORTED;
        PagedPrefillParams p{};
        p.ck = ck_q; p.cv = cv_q; p.kn = (const __half*)k_norms; p.vn = (const __half*)v_norms;
        p.block_table = block_table; p.lens = seq_lens; p.start = query_start; p.out = (__half*)out; p.partials = (float*)workspace; p.status = status;
        p.table_stride = table_stride; p.page_shift = shift; p.num_pages = num_pages; p.most_tokens = most;
        p.T = T; p.G = G; p.H = H; p.Hkv = Hkv; p.grp = grp; p.out_stride = out_stride; p.small_rows = m.small_rows;
        CUtensorMap tmQ, tmR;
        r = make_prefill_query_map(&tmQ, q, T, H, grp, qt, q_stride);
        if (r == TQ_OK) r = make_prefill_rows_map(&tmR, rotation, HEAD_DIM, HEAD_DIM);
        if (r != TQ_OK) return r;
        // CTAs: the most blocks that there can be, and where they may be cut, enough for their parts; where none may be there at all, two thirds of the SMs, so that
        // the launch for few rows starts on the others at once (4-bit 32/8 heads 32 x 1 to 5 behind 2000 to 4000 95 with all, 90; 12 x 1 to 20 behind 4000 78 / 81).
        const long long sms = std::min(device_props().sm_count, SPLIT_SMS), room = cut.mostly_small ? 2 * sms / 3 : sms;
        const dim3 grid((unsigned)std::max(ctas, std::min(room, ctas * cut.most_parts)));
        p.room = (int)std::min<long long>(grid.x, sms); p.most_parts = cut.most_parts;
        m.room = p.room; m.most_parts = cut.most_parts > 1 ? cut.most_parts : 0;
        if (cut.mt == 2) r = bits == 4 ? launch_paged_prefill<4, 2, false>(tmQ, tmR, p, grid, cs(s)) : launch_paged_prefill<2, 2, false>(tmQ, tmR, p, grid, cs(s));
        else if (cut.most_parts == 1) r = bits == 4 ? launch_paged_prefill<4, 1, false>(tmQ, tmR, p, grid, cs(s)) : launch_paged_prefill<2, 1, false>(tmQ, tmR, p, grid, cs(s));
        else r = bits == 4 ? launch_paged_prefill<4, 1, true>(tmQ, tmR, p, grid, cs(s)) : launch_paged_prefill<2, 1, true>(tmQ, tmR, p, grid, cs(s));
        if (r != TQ_OK) return r;
    }
    if (cut.small) {
        PagedRowsParams p{};
        p.ck = ck_q; p.cv = cv_q; p.kn = (const __half*)k_norms; p.vn = (const __half*)v_norms; p.q = (const __half*)q; p.rotation = (const __half*)rotation;
        p.block_table = block_table; p.lens = seq_lens; p.start = query_start; p.partials = small_sums; p.status = status;
        p.table_stride = table_stride; p.page_shift = shift; p.num_pages = num_pages; p.most_tokens = most;
        p.T = T; p.G = G; p.H = H; p.Hkv = Hkv; p.grp = grp; p.q_stride = q_stride; p.parts = cut.parts; p.row_blocks = (ROWS_MOST + 8 * cut.ncb - 1) / (8 * cut.ncb); p.behind = cut.large;
        p.by_request = (long long)G * most_small < T ? most_small : 0;
        p.part_tokens = p.by_request ? G * most_small : T;
        const long long ctas = (long long)Hkv * p.row_blocks * cut.parts * G;
        if (ctas >= (1ll << 31)) return TQ_ERR_UNSUPPORTED;
        const dim3 grid((unsigned)ctas);
        if (cut.ncb == 1) r = bits == 4 ? launch_rows<4, 1>(p, grid, cs(s)) : launch_rows<2, 1>(p, grid, cs(s));
        else if (cut.ncb == 3) r = bits == 4 ? launch_rows<4, 3>(p, grid, cs(s)) : launch_rows<2, 3>(p, grid, cs(s));
        else r = bits == 4 ? launch_rows<4, 2>(p, grid, cs(s)) : launch_rows<2, 2>(p, grid, cs(s));
        if (r != TQ_OK) return r;
        m.small_splits = cut.parts; m.part_tokens = p.part_tokens; m.by_request = p.by_request;
    }
    if (m.most_parts == 0 && m.small_splits == 0) return TQ_OK;
    // Rows of a request: 16 a CTA, which loop where a large one was cut: 16 CTAs per SM in all (as CTAs without work cost their turn), twice that where a large
    // request's would be few.  (us by 4, 8, 16, 32 of them, 4-bit 32/8 heads: 63 single tokens beside 64 behind 30000 221 / 221 / 198 / 187, 15 beside 200
    // behind 16000 218 / 198 / 186 / 183, 16 x 9 to 20 behind 600 to 1500, uncut, 37.9 / 38.9 / 39.7 / 41.4.)
    const long long most_rows = cut.large && m.most_parts ? (long long)T * H : (long long)std::min(T, most_small) * H, few = ((long long)std::min(T, most_small) * H + 15) / 16;
    const dim3 grid((unsigned)std::min<long long>((most_rows + 15) / 16, std::max<long long>({1, few, (cut.mostly_small ? 32 : 16) * device_props().sm_count / G})), (unsigned)G);
    return launch_kernel(paged_merge_kernel, grid, dim3(256), 0, cs(s), use_pdl(), m);
}

}  // extern "C"
