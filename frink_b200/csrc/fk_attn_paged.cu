// Attention over a paged KV cache: causal, grouped-query, with an optional window, first tokens that stay visible and a sink
// logit per head.  One new row a sequence (decode) or a few.
//
//   o = sum_j w_j v_j / (sum_j w_j + exp(sink)),  w_j = exp(scale q.k_j)  over the visible keys j
//
// kept as a running maximum m, a denominator l and unnormalised sums, so every key and value is read once; partial results of
// a split are joined by m.  All exponentials are powers of two (scale and log2 e go into q).
//
// Matrix products.  A warp takes 16 tokens of one KV head and 8 or 16 columns; a column is one (row, query head) pair of the
// group, so that all query heads of a KV head share one read of its keys.  Scores are K (16 tokens x 16 dims) times q
// (16 dims x 8 columns), outputs are V^T (16 dims x 16 tokens) times w (16 tokens x 8 columns), both mma.m16n8k16 with f32
// sums.  Which dims a lane's 16 bytes hold is free as long as both operands agree, so the order of dims is permuted instead
// of the data.  The scores' fragment becomes the weights' operand by a transposition of 8 x 8 blocks inside the warp (movmatrix).
//
// Memory.  16 tokens of one head are one contiguous piece of a page.  Every warp keeps a ring of its own in shared memory and
// fills it with asynchronous copies a step (32 tokens) ahead, keys and values apart, so that no warp waits for another and a
// step's latency is covered by the step before it and by the SM's other warps.  The copies place 16-byte pieces so that the
// operand reads hit every bank once.  8 x 4000 tokens of 24/8 heads of 128 in bf16: loads into registers 42.9 us, rings 37.9.
//
// Precision.  The cache's 16-bit values are exact operands.  q and w are f32 and are split into parts of the cache's type:
// three bf16 parts hold all 24 bits; two f16 parts hold 22, their range kept by a power of two per column of q and by a
// factor 2^14 on w.  f32 pages are split like q into three bf16 parts and the six products above 2^-24 are kept.  The tensor
// cores' own running sums are cut off rather than rounded, which over thousands of tiles adds up to a bias, so a product of
// a few steps starts from zero and joins the running sum in an ordinary, rounded addition.
//
// Work.  The keys of every (sequence, block of columns, KV head) are cut into units of 128 tokens (32 a warp; f32: 64) and all
// units, one after another, are dealt out in equal runs to the CTAs of one grid, so that ragged lengths keep every SM busy and
// the grid does not depend on lengths that only the device knows.  An item's way in (pages' numbers, q) and out (sums of the
// warps) takes about a unit's time and is dealt out like one: 500 sequences of 1 to 600 tokens, 8 KV heads, 155 us without, 125
// with (one row's own kernel: 113).  A run's first and last item may be shared with other CTAs: their partial sums go to a record of the CTA; the CTA that
// arrives last joins up to eight of them in one trip to memory, more in groups of about the square root of their number (131071
// tokens, 55 records an item: one CTA for all 57.2 us, groups 51.3).
//
// Bound by HBM where sequences are long, by its way in and out (some 10 us: launch, entries, page numbers, first copies, join)
// where they are short.  B200: 64 sequences of 250 to 16000 tokens, window 4096, 32/4 heads of 128 in bf16, 84 us = 5.7 TB/s;
// 131071 tokens, 64/8 heads of 64 in f16, 50.7 us = 5.3 TB/s, in f32 91 us = 5.9 TB/s; 8 x 4000 as above 28.6 us = 4.6 TB/s, in
// f32 51.4 us = 5.1 TB/s; 8 x 64000 6.4 TB/s; 17 tokens in f32 5.7 us.  (A plain copy moves 6.55 TB/s.)  Registers: three CTAs an
// SM leave 168 a thread (two, with 16 columns: 255), where one row's variants spill 44 bytes for heads of 128 in f16 and f32, 56
// with 16 columns in bf16, the others (almost) none; several rows' up to 76.
#include "fk_paged.cuh"

#include <type_traits>

using namespace fk_paged;

namespace {

constexpr int WARPS = 4;
// (sequence, block of columns) pairs that are dealt out in runs; where there are more, each (pair, KV head) has a CTA.  The deal
// costs a scan of the pairs by every CTA and keeps one long sequence from outlasting the others; 512 pairs dealt / 513 with CTAs
// of their own, us: 100 tokens and 8 KV heads 66 / 57, 1000 and 8 330 / 306, 1000 and 1 52 / 60, 4000 and 1 175 / 206; 500
// sequences of very different lengths (mean 8000) and 2 KV heads 631 / 1078.
constexpr int MAX_ENTRIES = 512;
constexpr int MAX_CTAS = 640;              // of a grid that shares items: three counters each
static_assert(3 * MAX_CTAS * sizeof(unsigned) <= WS_COUNTERS, "");
constexpr int FEW = 8;                     // records that are read together
constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
    const void* data;                      // the layer's pages
    const int *table, *lens, *n_new;
    const float *q, *sinks;
    float* out;
    unsigned* cnt;
    float* rec;
    int* err;
    float scale;
    int q_ld, rows, n_seqs, n_heads, n_kv, group, head_dim, page, log_page, n_pages, max_pages, window, first, n_cb, whole;
};

// ---- operand types
template <int KIND> struct Kind;
template <> struct Kind<KIND_F16> { static constexpr int Q = 2; };
template <> struct Kind<FK_BF16> { static constexpr int Q = 3; };
template <> struct Kind<KIND_F32> { static constexpr int Q = 3; };

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// (lo, hi) as parts: parts[0] the nearest pair of the type, parts[1] the nearest to what is left, ...
template <int KIND> __device__ __forceinline__ void split_pair(float lo, float hi, uint32_t* parts) {
    if (KIND == KIND_F16) {
        parts[0] = pack_f16(lo, hi);
        const __half2 h = *(const __half2*)&parts[0];
        parts[1] = pack_f16(lo - __low2float(h), hi - __high2float(h));
    } else {
        parts[0] = pack_bf16(lo, hi);
        lo -= __uint_as_float(parts[0] << 16);
        hi -= __uint_as_float(parts[0] & 0xffff0000u);
        parts[1] = pack_bf16(lo, hi);
        lo -= __uint_as_float(parts[1] << 16);
        hi -= __uint_as_float(parts[1] & 0xffff0000u);
        parts[2] = pack_bf16(lo, hi);
    }
}
template <int KIND> __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (KIND == KIND_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = a b: the same from zero (the sums start in the zero register)
template <int KIND> __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if (KIND == KIND_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// four 8 x 8 blocks, transposed: operand registers of 16 dims x 16 tokens from tokens' rows
__device__ __forceinline__ void ldsm_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float pow2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// a word of values with zeros in the place of what is not finite
template <int KIND> __device__ __forceinline__ uint32_t finite(uint32_t w) {
    constexpr uint32_t EXP = KIND == KIND_F32 ? 0x7f800000u : KIND == KIND_F16 ? 0x7c00u : 0x7f80u;      // a value's exponent
    if (KIND == KIND_F32) return (w & EXP) == EXP ? 0u : w;
    return w & (((w & EXP) == EXP ? 0u : 0xffffu) | ((w >> 16 & EXP) == EXP ? 0u : 0xffff0000u));
}

// ---- which keys an item sees: those below `hi`, in tiles of 16: [0, na) and then [b0, ...)
struct Span {
    int n;          // rows of the sequence
    int base;       // its length before them
    int lo;         // the oldest key of the window of the block's first row (0: no window)
    int hi;         // keys below this
    int na, b0, tiles;
};
// n: the sequence's rows, 0 where it would outgrow its table row
__device__ __forceinline__ int2 rows_of(const AttnArgs& a, int s, bool raise) {
    const int n = a.n_new ? min(max(a.n_new[s], 0), a.rows) : a.rows, base = a.lens[s];
    if (base >= 0 && (long long)base + n <= (long long)a.max_pages * a.page) return make_int2(base, n);
    if (raise && n > 0) fk_raise(a.err, 95);
    return make_int2(base, 0);
}
template <int COLS, bool ONE> __device__ __forceinline__ Span span_of(const AttnArgs& a, int2 base_n, int cb) {
    Span r;
    r.base = base_n.x;
    r.n = base_n.y;
    // one row: no division (a block of columns behind the group's has no row)
    const int row0 = ONE ? (cb * COLS < a.group ? 0 : 1) : cb * COLS / a.group;
    const int row1 = min(ONE ? 0 : (cb * COLS + COLS - 1) / a.group, r.n - 1);
    r.lo = r.hi = r.na = r.b0 = r.tiles = 0;
    if (row1 < row0) return r;                         // no real row in the block
    r.hi = r.base + row1 + 1;
    r.lo = a.window > 0 ? max(0, r.base + row0 + 1 - a.window) : 0;
    r.b0 = r.lo >> 4;
    r.na = (min(a.first, r.lo) + 15) >> 4;
    if (r.na >= r.b0) r.na = r.b0 = 0;
    r.tiles = r.na + ((r.hi + 15) >> 4) - r.b0;
    return r;
}

// A step of a warp is SUB tiles of 16 tokens (each in a page of its own, perhaps).  16-byte piece c of a tile's token r lies at
// c ^ swizzle(r): a read of K takes 4 pieces of 2 tokens at a time (f32: 4 even pieces of 2 tokens), one of V the same piece of
// 8 tokens (f32: 2 even pieces of 4 tokens), and with these the 8 addresses fall into 8 different groups of banks.
// A warp's ring is 16 KB whatever the type, so that an SM holds three CTAs: bytes in flight cover HBM's latency several times.
template <int KIND, int HDP> struct Ring {
    static constexpr int E = KIND == KIND_F32 ? 4 : 2;
    static constexpr int SUB = KIND == KIND_F32 ? 1 : 2;
    static constexpr int TILE = 16 * HDP * E;                              // bytes of 16 tokens' keys (or values)
    static constexpr int STAGES = 16384 / (2 * SUB * TILE);
    __host__ __device__ static constexpr int swz_k(int r) { return KIND == KIND_F32 ? r & 1 : (r & 1) << 2; }
    __host__ __device__ static constexpr int swz_v(int r) { return KIND == KIND_F32 ? ((r >> 1) & 1) | (r & 4) : r & 7; }
};

template <int KIND, int HDP, int NT> struct Smem {
    static constexpr int PITCH = HDP + 4;              // floats between columns of a warp's sums: stores hit every bank once
    static_assert(16384 >= NT * 8 * PITCH * 4, "a warp's sums take its ring's place at the end of an item");
    unsigned char ring[WARPS][16384];
    uint4 q[NT][HDP / 32][Kind<KIND>::Q][32];          // q's operand registers, part by part
    float qscale[NT * 8];                              // 2^-e of a column whose q was scaled by 2^e (f16)
    float m[WARPS][NT * 8], l[WARPS][NT * 8];
    int start[MAX_ENTRIES + 1];                        // first unit of every (sequence, block of columns)
    int part[33];
    int last;
};

// EXACT: heads of HDP, else shorter ones (their missing pieces are zeros).  ONE: one row a sequence, whose columns all see the same
// keys.  Us with a kernel for both / of its own: 512 x 100 tokens, bf16, 73.5 / 65.8, 8 x 4000 30.1 / 29.1, 17 tokens in f32 6.3 / 5.7.
template <int KIND, int HDP, bool EXACT, int NT, bool ONE>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 3 : 2) attn_paged_kernel(const AttnArgs a) {
    pdl_sync();
    constexpr int COLS = 8 * NT, KB = HDP / 32, VB = HDP / 64, QP = Kind<KIND>::Q;
    using R = Ring<KIND, HDP>;
    constexpr int E = R::E, SUB = R::SUB, STAGES = R::STAGES, ROWB = HDP * E, TILE = R::TILE, PITCH = Smem<KIND, HDP, NT>::PITCH;
    constexpr int STEP = WARPS * SUB;                              // tiles of a unit
    constexpr float SHIFT = KIND == KIND_F16 ? 14.0f : 0.0f;       // weights are 2^SHIFT times exp(score - m)
    extern __shared__ __align__(128) unsigned char smem_raw[];
    Smem<KIND, HDP, NT>& sm = *reinterpret_cast<Smem<KIND, HDP, NT>*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int hd = EXACT ? HDP : a.head_dim, n_e = a.n_seqs * a.n_cb;
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(sm.ring[warp]);
    float* const sum_o = reinterpret_cast<float*>(sm.ring[warp]);          // [COLS][PITCH] at the end of an item

    // ---- this CTA's run of slots [u, u_end): an item has one for its way in and out and one for each unit.  `start` of entry e:
    // slots before it (per KV head), times n_kv in the global order.
    // Up to 32 entries are scanned by every warp for itself, without a barrier; lane e keeps entry e.
    auto slots = [](const Span& sp) { return sp.tiles == 0 ? 0 : (sp.tiles + STEP - 1) / STEP + 1; };
    const bool few = n_e <= 32;
    int2 lane_rows = make_int2(0, 0);
    int lane_start = 0x7fffffff;
    int u, u_end, chunk;
    if (a.whole) {                                                 // one item a CTA: blockIdx.x = entry * n_kv + kv head
        u = 0;
        u_end = 1;
        chunk = 1;
    } else {
        int total = 0;
        if (few) {
            int units = 0;
            if (lane < n_e) {
                const int s = a.n_cb == 1 ? lane : lane / a.n_cb;
                lane_rows = rows_of(a, s, blockIdx.x == 0 && warp == 0);
                units = slots(span_of<COLS, ONE>(a, lane_rows, lane - s * a.n_cb));
            }
            int x = units;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane < n_e) lane_start = x - units;
            total = __shfl_sync(0xffffffffu, x, 31);
        } else {
            for (int e0 = 0; e0 < n_e; e0 += WARPS * 32) {
                const int e = e0 + tid;
                const int units = e < n_e ? slots(span_of<COLS, ONE>(a, rows_of(a, e / a.n_cb, blockIdx.x == 0), e % a.n_cb)) : 0;
                int sum;
                const int at = block_prefix(units, sm.part, &sum);
                if (e < n_e) sm.start[e] = total + at;
                total += sum;
                __syncthreads();
            }
        }
        const long long all = (long long)total * a.n_kv;
        if (all > 0x3fffffffLL) {                                  // no cache holds that many; table rows that share pages could claim it
            if (blockIdx.x == 0 && tid == 0) fk_raise(a.err, 95);
            return;
        }
        chunk = (int)((all + gridDim.x - 1) / gridDim.x);
        const long long b = (long long)blockIdx.x * chunk;
        u = (int)(b < all ? b : all);
        u_end = (int)(b + chunk < all ? b + chunk : all);
    }
    const int u_begin = u;

    while (u < u_end) {
        int e, kvh, i0, i1, first = 0, units, start = 0;           // units [i0, i1) of the item, the slot of its first unit
        int2 rows;
        if (a.whole) {
            e = blockIdx.x / a.n_kv;
            kvh = blockIdx.x % a.n_kv;
            rows = rows_of(a, e / a.n_cb, tid == 0);
        } else if (few) {                                          // the last entry that starts at or before u
            e = 31 - __clz(__ballot_sync(0xffffffffu, (long long)lane_start * a.n_kv <= u));
            start = __shfl_sync(0xffffffffu, lane_start, e);
            rows = make_int2(__shfl_sync(0xffffffffu, lane_rows.x, e), __shfl_sync(0xffffffffu, lane_rows.y, e));
        } else {
            int lo = 0, hi = n_e - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((long long)sm.start[mid] * a.n_kv <= u) lo = mid; else hi = mid - 1;
            }
            e = lo;
            start = sm.start[e];
            rows = rows_of(a, e / a.n_cb, false);
        }
        const int s = a.n_cb == 1 ? e : e / a.n_cb, cb = e - s * a.n_cb;
        const Span sp = span_of<COLS, ONE>(a, rows, cb);
        units = (sp.tiles + STEP - 1) / STEP;
        if (a.whole) {
            if (units == 0) return;
            i0 = 0;
            i1 = units;
            u = 1;
        } else {
            kvh = (u - start * a.n_kv) / (units + 1);
            first = start * a.n_kv + kvh * (units + 1) + 1;
            i0 = max(0, u - first);
            i1 = min(units, u_end - first);
            u = first + i1;
            if (i1 <= i0) break;                                   // the run ends before the item's first unit
        }

        // ---- the warp's steps: unit i0 + j, its tiles SUB (4 (i0 + j) + warp) and on of the item's list
        const int* tab = a.table + (size_t)s * a.max_pages;
        const uint32_t tok_bytes = hd * E;
        const size_t head_bytes = (size_t)a.page * tok_bytes;
        const char* const heads = (const char*)a.data + (size_t)kvh * head_bytes;
        const size_t half_bytes = (size_t)a.n_kv * head_bytes;     // a page's keys (or values)
        const int n_steps = max(0, min(i1, ((sp.tiles + SUB - 1) / SUB - warp + WARPS - 1) / WARPS) - i0);
        constexpr int NO_KEY = 0x7fffff00;                         // a tile behind the last one: no column sees it
        auto tile_key = [&](int j, int u) {                        // first key of a tile
            const int x = ((i0 + j) * WARPS + warp) * SUB + u;
            return x >= sp.tiles ? NO_KEY : (x < sp.na ? x : x - sp.na + sp.b0) << 4;
        };
        auto page_of = [&](int j, int u) {                         // its page, not looked at before the copy needs it
            const int k = j < n_steps ? tile_key(j, u) : NO_KEY;
            return k == NO_KEY ? 0 : tab[k >> a.log_page];
        };
        auto request = [&](auto values, int j, const int* pg) {    // starts the copy of a step's keys or values
            constexpr int V = decltype(values)::value;
            if (j < n_steps) {
#pragma unroll
                for (int u = 0; u < SUB; u++) {
                    const int k = tile_key(j, u);
                    if (k == NO_KEY) continue;
                    int page = pg[u];
                    if (page < 0 || page >= a.n_pages) {
                        if (lane == 0) fk_raise(a.err, 97);
                        page = 0;
                    }
                    const char* src = heads + (size_t)(2 * (uint32_t)page + V) * half_bytes + (uint32_t)(k & (a.page - 1)) * tok_bytes;
                    const uint32_t dst = ring + (((j % STAGES) * 2 + V) * SUB + u) * TILE;
                    constexpr int CH = ROWB / 16;
#pragma unroll
                    for (int i = 0; i < TILE / 512; i++) {
                        const int r = i * (32 / CH) + lane / CH, c = lane % CH;
                        const uint32_t at = r * ROWB + ((c ^ (V ? R::swz_v(r) : R::swz_k(r))) << 4);
                        if (EXACT) copy16(dst + at, src + (i * 32 + lane) * 16);
                        else if (c * 16 < tok_bytes) copy16(dst + at, src + r * tok_bytes + c * 16);
                    }
                }
            }
            copy_commit();
        };
        using Keys = std::integral_constant<int, 0>;
        using Values = std::integral_constant<int, 1>;

        __syncthreads();                                           // the previous item's shared memory is read
        if (!EXACT) {
            for (int i = lane; i < 16384 / 16; i += 32) reinterpret_cast<uint4*>(sm.ring[warp])[i] = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
        // The first pages' numbers and q are asked for ahead of the first copies, behind which they would queue.
        int pgs[STAGES][SUB];
#pragma unroll
        for (int j = 0; j < STAGES; j++)
#pragma unroll
            for (int u = 0; u < SUB; u++) pgs[j][u] = page_of(j, u);
        // q of the item's columns: scaled, split into parts, in operand registers' order.  A warp takes 32 dims of 8 columns at a
        // time (f16: all dims are read for the column's maximum).
        constexpr int QL = KIND == KIND_F16 ? KB : 1;
        auto q_load = [&](int x, float4 (&v)[QL][2]) {
            const int n = x % NT, kb = x / NT;
            const int c = cb * COLS + n * 8 + g, row = ONE ? (c < a.group ? 0 : 1) : c / a.group, h = kvh * a.group + (c - row * a.group);
            const float* qr = a.q + ((size_t)s * a.rows + row) * a.q_ld + (size_t)h * hd;
#pragma unroll
            for (int k = 0; k < QL; k++) {
                const int d = 32 * (QL == 1 ? kb : k) + 8 * t;
                v[k][0] = v[k][1] = make_float4(0, 0, 0, 0);
                if (row < sp.n && d < hd) {
                    v[k][0] = *(const float4*)(qr + d);
                    v[k][1] = *(const float4*)(qr + d + 4);
                }
            }
        };
        auto q_store = [&](int x, float4 (&v)[QL][2]) {
            const int n = x % NT, kb = x / NT;
            const float sl = a.scale * LOG2E;
            float4 y = v[0][0], z = v[0][1];
            float f = sl;
            if (KIND == KIND_F16) {
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < QL; k++) {
                    const float4 p = v[k][0], r = v[k][1];
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(p.x), fabsf(p.y)), fmaxf(fabsf(p.z), fabsf(p.w))));
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(r.x), fabsf(r.y)), fmaxf(fabsf(r.z), fabsf(r.w))));
                    if (k == kb) { y = p; z = r; }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * fabsf(sl);
                // 2^e with top * 2^e in [2^13, 2^14): no part leaves f16's range, and the low part keeps its bits
                int ex = top > 0.0f && top < INFINITY ? 13 - (int)((__float_as_uint(top) >> 23) & 255) + 127 : 0;
                ex = max(-100, min(100, ex));
                f = __uint_as_float((uint32_t)(127 + ex) << 23);
                y.x *= sl; y.y *= sl; y.z *= sl; y.w *= sl;
                z.x *= sl; z.y *= sl; z.z *= sl; z.w *= sl;
                if (t == 0 && kb == 0) sm.qscale[n * 8 + g] = __uint_as_float((uint32_t)(127 - ex) << 23);
            }
            uint32_t p[4][3];
            split_pair<KIND>(y.x * f, y.y * f, p[0]);
            split_pair<KIND>(y.z * f, y.w * f, p[1]);
            split_pair<KIND>(z.x * f, z.y * f, p[2]);
            split_pair<KIND>(z.z * f, z.w * f, p[3]);
#pragma unroll
            for (int k = 0; k < QP; k++) sm.q[n][kb][k][lane] = make_uint4(p[0][k], p[1][k], p[2][k], p[3][k]);
        };
        float4 qv[QL][2];
        if (warp < NT * KB) q_load(warp, qv);
#pragma unroll
        for (int j = 0; j < STAGES; j++) {
            request(Keys{}, j, pgs[j]);
            request(Values{}, j, pgs[j]);
        }
        if (warp < NT * KB) q_store(warp, qv);
        for (int x = warp + WARPS; x < NT * KB; x += WARPS) {
            q_load(x, qv);
            q_store(x, qv);
        }
        __syncthreads();

        // ---- this lane's columns: 2t and 2t + 1 of every block of 8
        int p_c[NT][2];                                            // position of the column's row; -1: no such column
        float cs[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int c = cb * COLS + n * 8 + 2 * t + k, row = ONE ? (c < a.group ? 0 : 1) : c / a.group;
                p_c[n][k] = row < sp.n ? sp.base + row : -1;
                cs[n][k] = KIND == KIND_F16 ? sm.qscale[n * 8 + 2 * t + k] : 1.0f;
            }
        // its first and last row's positions
        const int p_min = sp.base + (ONE ? 0 : cb * COLS / a.group), p_max = sp.hi - 1;
        float m[NT][2], l[NT][2], o[NT][VB * 4][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < VB * 4; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        }

        // operand addresses: K token g, dims 32 kb + 8 t; V token lane % 8 (+ 8), dims 16 d (+ 8) (f32: token 2 t, dims 64 vb + 8 g)
        const uint32_t k_at = ring + g * ROWB;
        const uint32_t v_at = ring + SUB * TILE +
                              (KIND == KIND_F32 ? 2 * t * ROWB : ((lane & 7) + 8 * (lane >> 4)) * ROWB + ((((lane >> 3) & 1) ^ (lane & 7)) << 4));
        // keys that a row of the block sees, and that every one does
        auto some_see = [&](int k) { return k <= p_max && (a.window <= 0 || k > p_min - a.window || k < a.first); };
        auto all_see = [&](int k) { return k <= p_min && (a.window <= 0 || k > p_max - a.window || k < a.first); };
        bool odd = false;                                          // a value that is not finite and that some columns see
        for (int j = 0; j < n_steps; j++) {
            const uint32_t stage = (j % STAGES) * 2 * SUB * TILE;
            int key0[SUB], pg_next[SUB];
            bool edge = false;
#pragma unroll
            for (int u = 0; u < SUB; u++) {
                key0[u] = tile_key(j, u);
                pg_next[u] = page_of(j + STAGES, u);
                // a tile that reaches over the newest key or the window's start
                edge = edge || key0[u] + 15 > p_min || (a.window > 0 && key0[u] <= p_max - a.window && key0[u] + 15 >= a.first);
            }
            copy_wait<2 * STAGES - 1>();
            __syncwarp();
            // scores
            float sc[SUB][NT][4];
#pragma unroll
            for (int u = 0; u < SUB; u++)
#pragma unroll
                for (int kb = 0; kb < KB; kb++) {
                    // two steps of 16 dims: registers 0, 1 and 2, 3 of both rows' pieces
                    uint32_t ka[KIND == KIND_F32 ? 3 : 1][2][4];
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const uint32_t row = k_at + stage + u * TILE + 8 * r * ROWB;
                        if (KIND == KIND_F32) {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const uint4 x = lds16(row + (((8 * kb + 2 * t + h) ^ R::swz_k(g)) << 4));
                                uint32_t p[3], q[3];
                                split_pair<FK_BF16>(__uint_as_float(x.x), __uint_as_float(x.y), p);
                                split_pair<FK_BF16>(__uint_as_float(x.z), __uint_as_float(x.w), q);
#pragma unroll
                                for (int k = 0; k < 3; k++) {
                                    ka[KIND == KIND_F32 ? k : 0][h][r] = p[k];
                                    ka[KIND == KIND_F32 ? k : 0][h][r + 2] = q[k];
                                }
                            }
                        } else {
                            const uint4 x = lds16(row + (((4 * kb + t) ^ R::swz_k(g)) << 4));
                            ka[0][0][r] = x.x;
                            ka[0][0][r + 2] = x.y;
                            ka[0][1][r] = x.z;
                            ka[0][1][r + 2] = x.w;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float x[4];
#pragma unroll
                        for (int k = QP - 1; k >= 0; k--) {        // the small parts first
                            const uint4 qv = sm.q[n][kb][k][lane];
#pragma unroll
                            for (int kk = (KIND == KIND_F32 ? 2 - k : 0); kk >= 0; kk--) {
                                if (k == QP - 1 && kk == (KIND == KIND_F32 ? 2 - k : 0)) mma0<KIND>(x, ka[kk][0], qv.x, qv.y);
                                else mma<KIND>(x, ka[kk][0], qv.x, qv.y);
                                mma<KIND>(x, ka[kk][1], qv.z, qv.w);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++) sc[u][n][k] = kb == 0 ? x[k] : sc[u][n][k] + x[k];
                    }
                }
            __syncwarp();
            request(Keys{}, j + STAGES, pg_next);
            if (KIND == KIND_F16) {
#pragma unroll
                for (int u = 0; u < SUB; u++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int k = 0; k < 4; k++) sc[u][n][k] *= cs[n][k & 1];
            }
            if (edge) {
#pragma unroll
                for (int u = 0; u < SUB; u++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int x = key0[u] + g + 8 * (k >> 1), p = p_c[n][k & 1];
                            const bool vis = x <= p && (a.window <= 0 || x > p - a.window || x < a.first);
                            if (!vis) sc[u][n][k] = -INFINITY;
                        }
            }
            // a new maximum anywhere in the warp: find it and rescale (rare once a sequence is under way)
            float top[NT][2];
            bool up = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float x = fmaxf(sc[0][n][k], sc[0][n][2 + k]);
                    if (SUB == 2) x = fmaxf(x, fmaxf(sc[SUB - 1][n][k], sc[SUB - 1][n][2 + k]));
                    top[n][k] = x;
                    up = up || x > m[n][k];
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        float x = fmaxf(top[n][k], m[n][k]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float corr = m[n][k] == -INFINITY ? 0.0f : pow2(m[n][k] - x);
                        m[n][k] = x;
                        l[n][k] *= corr;
#pragma unroll
                        for (int d = 0; d < VB * 4; d++) {
                            o[n][d][k] *= corr;
                            o[n][d][2 + k] *= corr;
                        }
                    }
            }
            // weights, as parts in the layout of the second product's operand
            uint32_t wp[SUB][NT][QP][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float m0 = m[n][0] == -INFINITY ? 0.0f : m[n][0] - SHIFT, m1 = m[n][1] == -INFINITY ? 0.0f : m[n][1] - SHIFT;
#pragma unroll
                for (int u = 0; u < SUB; u++) {
                    const float w0 = pow2(sc[u][n][0] - m0), w1 = pow2(sc[u][n][1] - m1), w2 = pow2(sc[u][n][2] - m0), w3 = pow2(sc[u][n][3] - m1);
                    l[n][0] += w0 + w2;
                    l[n][1] += w1 + w3;
                    uint32_t a0[3], a1[3];
                    split_pair<KIND>(w0, w1, a0);
                    split_pair<KIND>(w2, w3, a1);
#pragma unroll
                    for (int k = 0; k < QP; k++) {
                        wp[u][n][k][0] = transposed(a0[k]);
                        wp[u][n][k][1] = transposed(a1[k]);
                    }
                }
            }
            copy_wait<2 * STAGES - 1>();
            __syncwarp();
            if (edge) {
                // Values that no column sees become zeros, whatever they are (stale memory, NaN): they must not meet a weight of 0.
                // So do those that are not finite where only some columns see them, which get them at the end.
                const uint32_t vals = ring + stage + SUB * TILE;
                for (int x = lane; x < SUB * TILE / 16; x += 32) {
                    const int r = x / (ROWB / 16), k = (SUB == 2 && r >= 16 ? key0[SUB - 1] : key0[0]) + (r & 15);
                    if (!some_see(k)) {
                        sts16(vals + x * 16, make_uint4(0, 0, 0, 0));
                    } else if (!ONE && !all_see(k)) {
                        const uint4 y = lds16(vals + x * 16), z = make_uint4(finite<KIND>(y.x), finite<KIND>(y.y), finite<KIND>(y.z), finite<KIND>(y.w));
                        if (y.x != z.x || y.y != z.y || y.z != z.z || y.w != z.w) {
                            sts16(vals + x * 16, z);
                            odd = true;
                        }
                    }
                }
                __syncwarp();
            }
            // o += V^T w
            auto block = [&](int d, uint32_t (&va)[SUB][KIND == KIND_F32 ? 3 : 1][4]) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float x[4];
#pragma unroll
                    for (int k = QP - 1; k >= 0; k--)
#pragma unroll
                        for (int u = 0; u < SUB; u++)
#pragma unroll
                            for (int kk = (KIND == KIND_F32 ? 2 - k : 0); kk >= 0; kk--) {
                                if (k == QP - 1 && u == 0 && kk == (KIND == KIND_F32 ? 2 - k : 0)) mma0<KIND>(x, va[u][kk], wp[u][n][k][0], wp[u][n][k][1]);
                                else mma<KIND>(x, va[u][kk], wp[u][n][k][0], wp[u][n][k][1]);
                            }
#pragma unroll
                    for (int k = 0; k < 4; k++) o[n][d][k] += x[k];
                }
            };
            if (KIND == KIND_F32) {
#pragma unroll
                for (int vb = 0; vb < VB; vb++) {
                    uint4 v[4][2];
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            v[r][h] = lds16(v_at + stage + ((r & 1) + 8 * (r >> 1)) * ROWB + (((2 * (8 * vb + g) + h) ^ R::swz_v(2 * t)) << 4));
#pragma unroll
                    for (int d = 0; d < 4; d++) {              // dims 64 vb + 8 g + 2 d and + 1
                        uint32_t va[SUB][KIND == KIND_F32 ? 3 : 1][4];
                        float x[4][2];
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const uint4 y = v[r][d >> 1];
                            x[r][0] = __uint_as_float(d & 1 ? y.z : y.x);
                            x[r][1] = __uint_as_float(d & 1 ? y.w : y.y);
                        }
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                uint32_t p[3];
                                split_pair<FK_BF16>(x[2 * h][k], x[2 * h + 1][k], p);
#pragma unroll
                                for (int q = 0; q < 3; q++) va[0][KIND == KIND_F32 ? q : 0][2 * h + k] = p[q];
                            }
                        block(vb * 4 + d, va);
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < VB * 4; d++) {             // dims 16 d + g and + 8
                    uint32_t va[SUB][KIND == KIND_F32 ? 3 : 1][4];
#pragma unroll
                    for (int u = 0; u < SUB; u++) ldsm_t(va[u][0], (v_at + stage + u * TILE) ^ (d << 5));
                    block(d, va);
                }
            }
            __syncwarp();
            request(Values{}, j + STAGES, pg_next);
        }
        copy_wait<0>();
        __syncwarp();

        // ---- join the warps
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float x = l[n][k];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) {
                    sm.m[warp][n * 8 + 2 * t + k] = m[n][k];
                    sm.l[warp][n * 8 + 2 * t + k] = x;
                }
#pragma unroll
                for (int d = 0; d < VB * 4; d++) {
                    float* dst = sum_o + (n * 8 + 2 * t + k) * PITCH;
                    if (KIND == KIND_F32) {
                        *(float2*)(dst + 64 * (d >> 2) + 8 * g + 2 * (d & 3)) = make_float2(o[n][d][k], o[n][d][2 + k]);
                    } else {
                        dst[16 * d + g] = o[n][d][k];
                        dst[16 * d + 8 + g] = o[n][d][2 + k];
                    }
                }
            }
        // Values that are not finite and that only some columns see (none in any sane model) are added by themselves: they spoil
        // the columns that see them.
        if (!ONE && __any_sync(0xffffffffu, odd)) {
            __syncwarp();
#pragma unroll 1
            for (int x = 0; x < n_steps * SUB * 16; x++) {
                const int key0 = tile_key(x / (SUB * 16), x / 16 % SUB), k = key0 + (x & 15);
                if (key0 == NO_KEY || !some_see(k) || all_see(k)) continue;
                const int pg = tab[k >> a.log_page];
                const char* src = heads + (size_t)(2 * (uint32_t)(pg < 0 || pg >= a.n_pages ? 0 : pg) + 1) * half_bytes + (uint32_t)(k & (a.page - 1)) * tok_bytes;
                for (int d = lane; d < hd; d += 32) {
                    const float y = KIND == KIND_F32 ? ((const float*)src)[d] : KIND == KIND_F16 ? fk_h2f(((const uint16_t*)src)[d])
                                                                                                 : __uint_as_float((uint32_t)((const uint16_t*)src)[d] << 16);
                    if (fabsf(y) < INFINITY) continue;
                    for (int c = 0; c < COLS; c++) {
                        const int row = (cb * COLS + c) / a.group, p = sp.base + row;
                        if (row < sp.n && k <= p && (a.window <= 0 || k > p - a.window || k < a.first)) sum_o[c * PITCH + d] += y;
                    }
                }
            }
        }
        __syncthreads();
        auto finish = [&](int c, int d, float M, float L, float4 O) {      // four dims of a column
            const int cc = cb * COLS + c, row = ONE ? (cc < a.group ? 0 : 1) : cc / a.group, h = kvh * a.group + (cc - row * a.group);
            if (row >= sp.n || d >= hd) return;
            // against a maximum far below the sink the sum overflows to infinity and the output is 0, as it should be
            if (a.sinks) L += M == -INFINITY ? 1.0f : pow2(a.sinks[h] * LOG2E - M + SHIFT);
            const float inv = 1.0f / L;
            *(float4*)(a.out + ((size_t)s * a.rows + row) * a.n_heads * hd + (size_t)h * hd + d) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
        };
        const bool direct = a.whole || (i0 == 0 && i1 == units);
        // a CTA's record 1 is the item that begins in its run and goes on behind it, record 0 the one that began before
        float* rec = a.rec + ((size_t)2 * blockIdx.x + (first >= u_begin ? 1 : 0)) * ATTN_RECORD;
        for (int x = tid; x < COLS * (HDP / 4); x += WARPS * 32) {
            const int c = x / (HDP / 4), d = 4 * (x % (HDP / 4));
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; w++) M = fmaxf(M, sm.m[w][c]);
            float L = 0.0f;
            float4 O = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = sm.m[w][c] == -INFINITY ? (sm.l[w][c] != sm.l[w][c] ? sm.l[w][c] : 0.0f) : pow2(sm.m[w][c] - M);
                const float4 v = *(const float4*)(reinterpret_cast<const float*>(sm.ring[w]) + c * PITCH + d);
                L += sm.l[w][c] * f;
                O.x += v.x * f; O.y += v.y * f; O.z += v.z * f; O.w += v.w * f;
            }
            if (direct) {
                finish(c, d, M, L, O);
            } else {
                *(float4*)(rec + c * 128 + d) = O;
                if (d == 0) {
                    rec[16 * 128 + c] = M;
                    rec[16 * 129 + c] = L;
                }
            }
        }
        if (direct) continue;

        // ---- join the records of CTAs [c0, c0 + n_rec).  Few: the last one to arrive takes them all.  More: groups of about the
        // square root of their number are joined into their first record by the group's last one, and those by the last group's.
        const int c0 = first / chunk, n_rec = (first + units - 1) / chunk - c0 + 1;
        // whether all n have arrived; a CTA's record goes out by way of the barrier and this release, the others' come in by the acquire
        auto arrive = [&](unsigned* cnt, int n) {
            __syncthreads();
            if (tid == 0) {
                unsigned before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(cnt) : "memory");
                sm.last = before == (unsigned)(n - 1);
                if (sm.last) *cnt = 0;
            }
            __syncthreads();
            return sm.last != 0;
        };
        // record 1 of the CTA in which the item begins, record 0 of the others
        auto slot = [&](int k) { return 2 * (c0 + k) + (k == 0 ? 1 : 0); };
        // records k0, k0 + step, ... (n of them) of four dims of a column, eight at a time
        auto gather = [&](int k0, int step, int n, int c, int d, float& M, float& L, float4& O) {
            M = -INFINITY;
            L = 0.0f;
            O = make_float4(0, 0, 0, 0);
            for (int b = 0; b < n; b += FEW) {
                float mk[FEW], lk[FEW], top = M;
                float4 v[FEW];
#pragma unroll
                for (int k = 0; k < FEW; k++) {
                    mk[k] = -INFINITY;
                    lk[k] = 0.0f;
                    v[k] = make_float4(0, 0, 0, 0);
                    if (b + k < n) {
                        const float* r = a.rec + (size_t)slot(k0 + (b + k) * step) * ATTN_RECORD;
                        mk[k] = __ldcg(r + 16 * 128 + c);
                        lk[k] = __ldcg(r + 16 * 129 + c);
                        v[k] = __ldcg((const float4*)(r + c * 128 + d));
                    }
                }
#pragma unroll
                for (int k = 0; k < FEW; k++) top = fmaxf(top, mk[k]);
                const float f0 = M == -INFINITY ? 1.0f : pow2(M - top);                  // nothing yet, or NaN, which stays
                L *= f0;
                O.x *= f0; O.y *= f0; O.z *= f0; O.w *= f0;
#pragma unroll
                for (int k = 0; k < FEW; k++) {
                    const float f = mk[k] == -INFINITY ? (lk[k] != lk[k] ? lk[k] : 0.0f) : pow2(mk[k] - top);
                    L += lk[k] * f;
                    O.x += v[k].x * f; O.y += v[k].y * f; O.z += v[k].z * f; O.w += v[k].w * f;
                }
                M = top;
            }
        };
        int per = FEW;
        while (per * per < n_rec) per++;
        const int groups = (n_rec + per - 1) / per;
        if (groups > 1) {
            const int g0 = ((int)blockIdx.x - c0) / per * per, n = min(per, n_rec - g0);
            if (!arrive(a.cnt + slot(g0), n)) continue;
            float* const to = a.rec + (size_t)slot(g0) * ATTN_RECORD;
            for (int x = tid; x < COLS * (HDP / 4); x += WARPS * 32) {
                const int c = x / (HDP / 4), d = 4 * (x % (HDP / 4));
                float M, L;
                float4 O;
                gather(g0, 1, n, c, d, M, L, O);
                *(float4*)(to + c * 128 + d) = O;                  // only this thread read this place
                if (d == 0) {
                    sm.m[0][c] = M;
                    sm.l[0][c] = L;
                }
            }
            __syncthreads();
            if (tid < COLS) {
                to[16 * 128 + tid] = sm.m[0][tid];
                to[16 * 129 + tid] = sm.l[0][tid];
            }
        }
        if (!arrive(a.cnt + 2 * MAX_CTAS + c0, groups > 1 ? groups : n_rec)) continue;
        for (int x = tid; x < COLS * (HDP / 4); x += WARPS * 32) {
            const int c = x / (HDP / 4), d = 4 * (x % (HDP / 4));
            float M, L;
            float4 O;
            gather(0, groups > 1 ? per : 1, groups > 1 ? groups : n_rec, c, d, M, L, O);
            finish(c, d, M, L, O);
        }
    }
}

template <int KIND, int HDP, bool EXACT, int NT, bool ONE> int launch_attn(fk_ctx* ctx, cudaStream_t st, AttnArgs a) {
    auto kern = attn_paged_kernel<KIND, HDP, EXACT, NT, ONE>;
    const size_t smem = sizeof(Smem<KIND, HDP, NT>);
    static thread_local int resident[64] = {};                     // CTAs an SM holds, by device
    int& per_sm = resident[ctx->device & 63];
    if (per_sm == 0) {
        FK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), FK_KERNEL);
        FK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared), FK_KERNEL);
        int n = 0;
        FK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, WARPS * 32, smem), FK_KERNEL);
        per_sm = n < 1 ? 1 : n > ATTN_CTAS_PER_SM ? ATTN_CTAS_PER_SM : n;
    }
    a.n_cb = (int)(((long long)a.rows * a.group + 8 * NT - 1) / (8 * NT));
    const long long entries = (long long)a.n_cb * a.n_seqs;
    if (entries * a.n_kv > 0x7fffffffLL) return fk_fail(FK_UNSUPPORTED, "attention_paged: %d rows of %d sequences", a.rows, a.n_seqs);
    // the deal counts slots in 32 bits, full table rows' too
    a.whole = entries > MAX_ENTRIES || entries * ((long long)a.max_pages * a.page / (16 * WARPS * Ring<KIND, HDP>::SUB) + 2) > 1 << 30;
    const int ctas = per_sm * ctx->sm_count;
    const unsigned grid = a.whole ? (unsigned)(entries * a.n_kv) : (unsigned)(ctas < MAX_CTAS ? ctas : MAX_CTAS);
    FK_CUDA(launch(kern, dim3(grid), dim3(WARPS * 32), smem, st, a), FK_LAUNCH);
    return FK_OK;
}

template <int KIND, bool ONE> int launch_kind(fk_ctx* ctx, cudaStream_t st, const AttnArgs& a) {
    // 16 columns a CTA read the keys once for twice the columns, with registers for two CTAs an SM instead of three.  Us with 16 /
    // with 8: 16 columns, 4 KV heads, 64 x 4000 tokens 114 / 171, 8 x 16000 67 / 87, 1 x 64000 49 / 42; 12 columns, 3 KV heads,
    // 64 x 4000 90 / 130.
    const bool wide = (long long)a.rows * a.group > 8;
    if (a.head_dim == 64) return wide ? launch_attn<KIND, 64, true, 2, ONE>(ctx, st, a) : launch_attn<KIND, 64, true, 1, ONE>(ctx, st, a);
    if (a.head_dim == 128) return wide ? launch_attn<KIND, 128, true, 2, ONE>(ctx, st, a) : launch_attn<KIND, 128, true, 1, ONE>(ctx, st, a);
    return wide ? launch_attn<KIND, 128, false, 2, ONE>(ctx, st, a) : launch_attn<KIND, 128, false, 1, ONE>(ctx, st, a);
}

template <int KIND> int launch_rows(fk_ctx* ctx, cudaStream_t st, const AttnArgs& a) {
    return a.rows == 1 ? launch_kind<KIND, true>(ctx, st, a) : launch_kind<KIND, false>(ctx, st, a);
}

}  // namespace

FK_EXPORT int fk_attention_paged(fk_ctx* ctx, void* stream, const fk_pages* p, int layer, const float* q_dev, int q_ld, int rows, const int* n_new_dev,
                                 int n_heads, float scale, int window, int first, const float* sinks_dev, float* out_dev) {
    int rc = check("attention_paged", ctx, p, layer);
    if (rc != FK_OK) return rc;
    if (!q_dev || !out_dev) return fk_fail(FK_INVALID, "attention_paged: null argument");
    if (window < 0 || first < 0) return fk_fail(FK_INVALID, "attention_paged: window %d, first %d", window, first);
    if (rows < 1 || n_heads < 1 || n_heads % p->n_kv || (long long)rows * p->n_seqs > 0x7fffffffLL || (long long)n_heads * p->head_dim > 0x7fffffffLL)
        return fk_fail(FK_UNSUPPORTED, "attention_paged: %d rows, %d/%d heads of %d", rows, n_heads, p->n_kv, p->head_dim);
    if (q_ld == 0) q_ld = n_heads * p->head_dim;
    if (q_ld < n_heads * p->head_dim || (q_ld & 3) || (((uintptr_t)q_dev | (uintptr_t)out_dev) & 15))
        return fk_fail(FK_INVALID, "attention_paged: rows must be 16-byte aligned, %d floats apart", q_ld);
    FkDeviceGuard g(ctx->device);
    AttnArgs a{(const char*)p->data_dev + (size_t)layer * page_bytes(p) * p->n_pages, p->table_dev, p->lens_dev, n_new_dev, q_dev, sinks_dev, out_dev,
               (unsigned*)p->ws_dev, (float*)((char*)p->ws_dev + WS_COUNTERS), ctx->err_flag, scale, q_ld, rows, p->n_seqs, n_heads, p->n_kv,
               n_heads / p->n_kv, p->head_dim, p->page, p->page == 16 ? 4 : p->page == 32 ? 5 : p->page == 64 ? 6 : 7, p->n_pages, p->max_pages, window, first, 0, 0};
    cudaStream_t st = (cudaStream_t)stream;
    if (fk_attn_prompt_takes(ctx, p, rows, n_heads))
        rc = fk_attn_prompt_launch(ctx, st, p, layer, q_dev, q_ld, rows, n_new_dev, n_heads, scale, window, first, sinks_dev, out_dev);
    else rc = p->kind == KIND_F32 ? launch_rows<KIND_F32>(ctx, st, a) : p->kind == KIND_F16 ? launch_rows<KIND_F16>(ctx, st, a) : launch_rows<FK_BF16>(ctx, st, a);
    if (rc != FK_OK) return rc;
    FK_CUDA(cudaGetLastError(), FK_LAUNCH);
    ctx->launches++;
    return FK_OK;
}
