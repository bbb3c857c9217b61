// Attention of a prompt's rows over a paged KV cache on the tensor cores (tcgen05): 16-bit pages, heads of up to 128.  The
// mathematics, the masks and the precision are those of fk_attn_paged.cu.
//
// An item is 128 (row, query head) pairs of one KV head -- 128 / group consecutive rows, so a short prompt still fills the
// tile -- and the visible keys in tiles of 64.  There is a CTA per SM, which goes through its items with the rings running on:
// the next item's first tiles and q are on their way while the current one ends (the last case below: 393 us, 430 with a CTA per
// item).  A tile:
//
//   S = q K^T          A = q's parts in tensor memory, B = a tile of K in shared memory, S in tensor memory (two or three buffers)
//   w = 2^(S - m)      a thread per row; its parts go back over S as the next product's A operand
//   O = w V            A = w's parts, B = the tile of V as it lies in memory (the major axis is its dims)
//   o = o c + O        in registers, every tile: the tensor core cuts its sums off instead of rounding them, and an O that stayed
//                      there lost 1.1e-7 of its size every 16 keys (2e-4 at 30000 keys, measured with values of one sign)
//
// bf16 takes three parts of q and w, f16 two (fk_attn_paged.cu says why that is f32 precision), so a product is three (two)
// products: the bound is the tensor cores' rate by that factor.  Per tile of 64 keys and 128 dims that is 1536 (1024) cycles of
// MMA against 512 of exponentials and some 700 issue slots a scheduler for the parts and the running output.
//
// Warps 0 to 7 are the softmax: a thread has a row and half of the tile's keys, and the halves exchange the row's maximum.
// (Two groups that take turns with a tile each need no exchange, but a tile is then twice as long between its scores and its
// weights, and that chain bounds the kernel: 4200 rows of 24/8 heads of 128, bf16, 398 us that way, 326 us this way, with a CTA
// per item.)  8 to 15 keep the running output, a thread per row and half of the
// dims.  16 loads tiles (a lane per page piece, TMA with 128-byte swizzle).  17 issues the products for S and 19 those for O, so
// that scores are made as soon as their buffer is free and not in turn with products that wait for weights.  18 looks over the
// values of tiles that not every row sees: a value that no row sees is zeroed in shared memory (stale memory may hold NaN); one
// that some rows see and that is not finite is zeroed too and added in plain f32 for the rows that see it.
//
// Measured (B200): 512 rows of 24/8 heads of 128, bf16, empty cache 23.5 us; 4200 rows 309 us = 351 TFLOP/s of the formula's
// operations, three times that of MMA, f16 267 us; 1001, 801, 601 and 401 rows after 2000 to 8000 tokens, window 2048, 64/8
// heads of 64, f16, 385 us.  What bounds it is a tile's chain from scores to weights (tensor pipe 25 %, issue slots 49 %): with
// one part of each product instead of two or three the last case gains 3 % and the bf16 one 6 %, without the exponentials and
// the parts' arithmetic 20 and 9 %.  An item alone is bound by its way in and out.
#include "fk_paged.cuh"
#include "fk_tc.cuh"

#include <type_traits>

using namespace fk_paged;
using namespace fk_tc;

namespace {

constexpr int KT = 64;                         // keys of a tile

constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t SPINS = 1u << 16;           // tests of a wait before it gives up, each of up to PARK nanoseconds
constexpr uint32_t PARK = 10000;

struct PromptArgs {
    CUtensorMap map;                           // the layer's pages as [tokens of all pages, halves and heads][head_dim]
    const void* data;
    const int *table, *lens, *n_new;
    const float *q, *sinks;
    float* out;
    int* err;
    float scale;
    int q_ld, rows, n_seqs, n_heads, n_kv, group, head_dim, page, log_page, n_pages, max_pages, window, first, rq, n_rb;
};

template <int KIND, int HD> struct Plan {
    static constexpr int QP = KIND == KIND_F16 ? 2 : 3;            // parts of q and of the weights
    static constexpr int TILE = KT * HD * 2;                       // bytes of a tile of K or V
    static constexpr int STAGES = HD == 64 ? 6 : 4;
    // warps: 8 of the softmax, 8 of the running output, then the four single ones
    static constexpr int OUT = 8, LOADER = 16, ISSUER_S = 17, LOOKER = 18, ISSUER_O = 19;
    static constexpr int THREADS = 32 * (LOADER + 4);
    // Tensor memory columns of a tile: S's 64 behind LEAD free ones; the parts of w's first half of the keys take the free ones
    // and S's first half, those of its second half what follows, so that S is never overwritten before it is read.
    static constexpr int SREG = QP * 32, LEAD = SREG - 64;
    // buffers of O and of S, as tensor memory allows: with two of O a product need not wait for the running output to take the
    // last one, with three of S not for the product whose operand it overwrites
    static constexpr int NO = HD == 64 ? 2 : 1;
    static constexpr int Q0 = 0, O0 = QP * HD / 2, S0 = O0 + NO * HD;
    static constexpr int NS = S0 + 4 * SREG <= 512 ? 4 : S0 + 3 * SREG <= 512 ? 3 : 2;
    static_assert(S0 + NS * SREG <= 512, "tensor memory");
};

template <int KIND, int HD> struct PromptSmem {
    using P = Plan<KIND, HD>;
    unsigned char k[P::STAGES][P::TILE];
    unsigned char v[P::STAGES][P::TILE];
    float stage[128 * HD];                     // rows of q and of the output on their way; between them the weights of a tile's values
                                               // that are not finite, [key][row] (-1: the row does not see it)
    float top[2][2][128];                      // a row's maximum over each half of the tile's keys, two tiles' worth
    float corr[8][128];                        // what the running output is multiplied with at the tile (mod 8)
    float fin[2][2][128];                      // denominator of each half's keys and the maximum (the same for both)
    unsigned long long odd_of[8];              // which of the tile's values are not finite (mod 8)
    unsigned long long odd[P::STAGES];         // the same, where the values lie
    unsigned long long kfull[P::STAGES], kfree[P::STAGES], vfull[P::STAGES], vfree[P::STAGES], vready[P::STAGES];
    unsigned long long sfull[P::NS], pfull[P::NS], oddfree, ofull[P::NO], ofree[P::NO], qfull, done[2];
    uint32_t tmem;
    int abort;
};

// 128 / group rows of a sequence and one KV head, and the keys they see: [0, 64 na) and [64 b0, hi)
struct Item {
    int kvh, s, row0, row1, base, hi, na, b0, n_tiles;
    __device__ __forceinline__ int p_min() const { return base + row0; }
    __device__ __forceinline__ int p_max() const { return hi - 1; }
    __device__ __forceinline__ int key(int j) const { return (j < na ? j : j - na + b0) * KT; }
    // whether some row does not see all of the tile
    __device__ __forceinline__ bool edge(const PromptArgs& a, int key0) const {
        return key0 + KT - 1 > p_min() || (a.window > 0 && key0 <= p_max() - a.window && key0 + KT - 1 >= a.first);
    }
};

// d (+)= a b: A in tensor memory.  Issued by one lane, inside `if (elected())`: the compiler then knows that one thread runs
// and keeps the operands in uniform registers.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0) : "memory");
}
// Whether the phase has completed; the hardware parks the warp until it has or PARK is over, so that a dozen waiting warps do not
// take issue slots and shared memory from the others.
__device__ __forceinline__ bool parked(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(PARK) : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// f32 sums of f16 or bf16 products; b_mn: B's major axis is N
__host__ __device__ constexpr uint32_t idesc_of(int kind, int m, int n, int b_mn) {
    return (1u << 4) | (kind == KIND_F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ float pow2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// two at a time: the last case 393 -> 386 us, f16 heads of 128 286 -> 276
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b), "l"(*(uint64_t*)&c));
    return *(float2*)&r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
    return *(float2*)&r;
}
// (lo, hi) rounded to a pair of the type; lo and hi become what is left
template <int KIND> __device__ __forceinline__ uint32_t take_part(float& lo, float& hi) {
    uint32_t r;
    float2 h;
    if (KIND == KIND_F16) {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        h = __half22float2(*(const __half2*)&r);
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        h = make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
    }
    const float2 left = fma2(h, make_float2(-1.0f, -1.0f), make_float2(lo, hi));
    lo = left.x;
    hi = left.y;
    return r;
}
template <int N> __device__ __forceinline__ void tm_ld(uint32_t addr, float* v) {
    static_assert(N == 16 || N % 32 == 0, "");
    if (N == 16) tc_ld16(addr, reinterpret_cast<uint32_t*>(v));
#pragma unroll
    for (int i = 0; i + 32 <= N; i += 32) tc_ld32(addr + i, reinterpret_cast<uint32_t*>(v) + i);
    tc_wait_ld();
    tc_ld_fence<N>(reinterpret_cast<uint32_t*>(v));
}

template <int KIND, int HD>
__global__ void __launch_bounds__((Plan<KIND, HD>::THREADS), 1) attn_prompt_kernel(const __grid_constant__ PromptArgs a) {
    using P = Plan<KIND, HD>;
    constexpr int QP = P::QP, STAGES = P::STAGES, NS = P::NS, NO = P::NO, HALF = HD / 2;
    constexpr float SHIFT = KIND == KIND_F16 ? 14.0f : 0.0f;
    extern __shared__ unsigned char smem_raw[];
    PromptSmem<KIND, HD>& sm = *reinterpret_cast<PromptSmem<KIND, HD>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), hd = a.head_dim;
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) {
            mbar_init(smem_u32(&sm.kfull[i]), 1);
            mbar_init(smem_u32(&sm.kfree[i]), 1);
            mbar_init(smem_u32(&sm.vfull[i]), 1);
            mbar_init(smem_u32(&sm.vfree[i]), 1);
            mbar_init(smem_u32(&sm.vready[i]), 1);
        }
        for (int i = 0; i < NS; i++) {
            mbar_init(smem_u32(&sm.sfull[i]), 1);
            mbar_init(smem_u32(&sm.pfull[i]), 8);
        }
        mbar_init(smem_u32(&sm.oddfree), 8);
        for (int i = 0; i < NO; i++) {
            mbar_init(smem_u32(&sm.ofull[i]), 1);
            mbar_init(smem_u32(&sm.ofree[i]), 8);
        }
        mbar_init(smem_u32(&sm.qfull), 16);
        mbar_init(smem_u32(&sm.done[0]), 1);
        mbar_init(smem_u32(&sm.done[1]), 1);
        sm.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // ---- this CTA's items, one after another: long ones (late rows) come first, every other round in reverse.  All warps go
    // through them for themselves; t0 counts tiles, by which the rings go on from one item to the next.
    const int n_items = a.n_rb * a.n_seqs * a.n_kv;
    auto item_at = [&](int i, Item& x) {
        const long long at = (long long)i * gridDim.x + (i & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (at >= n_items) return false;
        const unsigned it = (unsigned)at;
        x.kvh = it % (unsigned)a.n_kv;
        x.s = it / (unsigned)a.n_kv % (unsigned)a.n_seqs;
        x.row0 = (a.n_rb - 1 - (int)(it / ((unsigned)a.n_kv * a.n_seqs))) * a.rq;
        int n = a.n_new ? min(max(a.n_new[x.s], 0), a.rows) : a.rows;
        x.base = a.lens[x.s];
        if (x.base < 0 || (long long)x.base + n > (long long)a.max_pages * a.page) {
            if (tid == 0 && n > 0) fk_raise(a.err, 95);
            n = 0;
        }
        x.row1 = min(x.row0 + a.rq, n) - 1;
        x.hi = x.base + x.row1 + 1;
        const int lo = a.window > 0 ? max(0, x.base + x.row0 + 1 - a.window) : 0;
        x.b0 = lo / KT;
        x.na = (min(a.first, lo) + KT - 1) / KT;
        if (x.na >= x.b0) x.na = x.b0 = 0;
        x.n_tiles = __shfl_sync(0xffffffffu, x.row1 < x.row0 ? 0 : x.na + (x.hi + KT - 1) / KT - x.b0, 0);
        return true;
    };
    Item it;
    bool more = item_at(0, it);

    // Tensor memory is taken after the previous kernel is done with its own and before the next one may start: neither can
    // then hold what the other waits for.
    if (warp == P::ISSUER_S) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // a wait gives up after SPINS polls, or at once when another one of the CTA has given up; the CTA then runs to its end
    auto wait = [&](unsigned long long* bar, uint32_t parity) {
        const uint32_t b = smem_u32(bar);
        // the warp goes on together: what it does next stays uniform for the compiler, and operands in uniform registers
        for (uint32_t i = 0; i < SPINS; i++) {
            if (__all_sync(0xffffffffu, parked(b, parity))) return;
            if (__any_sync(0xffffffffu, *(volatile int*)&sm.abort)) return;
        }
        *(volatile int*)&sm.abort = 1;
        fk_raise(a.err, 63);
    };
    auto gave_up = [&] { return __any_sync(0xffffffffu, *(volatile int*)&sm.abort) != 0; };      // the same answer for the whole warp

    if (warp == P::LOADER) {
        // ---- loads: lane u takes the u-th page piece of a tile.  The page numbers of 32 pieces are read at once, a lane each and
        // a block of tiles ahead: a table lookup takes longer than a tile.
        const int log_piece = min(a.log_page, 6), log_pc = 6 - log_piece, n_pc = 1 << log_pc, ahead = 32 >> log_pc;
        int issued = 0;
        for (int i = 0, t0 = 0; more; t0 += it.n_tiles, more = item_at(++i, it)) {
            const Item& x = it;
            const int* const tab = a.table + (size_t)x.s * a.max_pages;
            auto pages_from = [&](int j0) {
                const int j = j0 + (lane >> log_pc);
                const int key = j < x.n_tiles ? x.key(j) + ((lane & (n_pc - 1)) << log_piece) : x.hi;
                return key < x.hi ? tab[key >> a.log_page] : -1;
            };
            int block = pages_from(0), next = pages_from(ahead);
            for (int j = 0; j < x.n_tiles; j++) {
                const int t = t0 + j, st = t % STAGES, in_block = j & (ahead - 1);
                if (j > 0 && in_block == 0) {
                    block = next;
                    next = pages_from(j + ahead);
                }
                const int key0 = x.key(j), key = key0 + (lane << log_piece);
                int pg = __shfl_sync(0xffffffffu, block, (in_block << log_pc) + (lane & (n_pc - 1)));
                const int pieces = min(n_pc, (x.hi - key0 + (1 << log_piece) - 1) >> log_piece);
                const bool mine = lane < pieces;
                if (mine && (pg < 0 || pg >= a.n_pages)) {
                    fk_raise(a.err, 97);
                    pg = 0;
                }
                const int y = ((2 * pg) * a.n_kv + x.kvh) * a.page + (key & (a.page - 1));
                if (t >= STAGES) wait(&sm.kfree[st], (t / STAGES - 1) & 1);
                if (t >= STAGES) wait(&sm.vfree[st], (t / STAGES - 1) & 1);
                if (gave_up()) break;
                if (lane == 0) {
                    mbar_expect_tx(smem_u32(&sm.kfull[st]), (pieces << log_piece) * HD * 2);
                    mbar_expect_tx(smem_u32(&sm.vfull[st]), (pieces << log_piece) * HD * 2);
                }
                __syncwarp();
                if (mine) {
#pragma unroll
                    for (int h = 0; h < HD / 64; h++)
                        tma_load_2d(smem_u32(sm.k[st]) + h * (KT * 128) + (lane << log_piece) * 128, &a.map, h * 64, y, smem_u32(&sm.kfull[st]));
#pragma unroll
                    for (int h = 0; h < HD / 64; h++)
                        tma_load_2d(smem_u32(sm.v[st]) + h * (KT * 128) + (lane << log_piece) * 128, &a.map, h * 64, y + a.n_kv * a.page, smem_u32(&sm.vfull[st]));
                }
                issued = t + 1;
            }
            if (gave_up()) break;
        }
        // every copy that was started has landed before the CTA ends
        for (int j = max(0, issued - STAGES); j < issued; j++) {
            const uint32_t par = (j / STAGES) & 1;
            for (uint32_t i = 0; i < SPINS && !parked(smem_u32(&sm.kfull[j % STAGES]), par); i++) {}
            for (uint32_t i = 0; i < SPINS && !parked(smem_u32(&sm.vfull[j % STAGES]), par); i++) {}
        }
    } else if (warp == P::ISSUER_S) {
        // ---- S = q K^T
        constexpr uint32_t ID_S = idesc_of(KIND, 128, KT, 0);
        const uint64_t k_desc = umma_desc(smem_u32(sm.k[0]));
        for (int i = 0, t0 = 0, done = 0; more && !gave_up(); t0 += it.n_tiles, more = item_at(++i, it)) {
            if (it.n_tiles == 0) continue;
            wait(&sm.qfull, done++ & 1);
            for (int t = t0; t < t0 + it.n_tiles && !gave_up(); t++) {
                const int st = t % STAGES, x = t - NS;
                // S takes the place of w of tile t - NS: products with different results may pass one another, so that one is waited for
                if (x >= 0) wait(&sm.vfree[x % STAGES], (x / STAGES) & 1);
                wait(&sm.kfull[st], (t / STAGES) & 1);
                tc_fence_after();
                const uint32_t d = tmem + P::S0 + (t % NS) * P::SREG + P::LEAD;
                const uint64_t b = k_desc + (uint32_t)(st * (P::TILE >> 4));
                if (elected()) {
#pragma unroll
                    for (int k = QP - 1; k >= 0; k--)              // the small parts first
#pragma unroll
                        for (int ks = 0; ks < HD / 16; ks++)
                            mma_ts(d, tmem + P::Q0 + k * HALF + ks * 8, b + (((ks >> 2) * (KT * 128) + (ks & 3) * 32) >> 4), ID_S, k < QP - 1 || ks > 0);
                    tc_commit(smem_u32(&sm.sfull[t % NS]));
                    tc_commit(smem_u32(&sm.kfree[st]));
                }
                __syncwarp();
            }
        }
        // tensor memory is given back only when no product is under way
        if (elected()) tc_commit(smem_u32(&sm.done[0]));
        __syncwarp();
        for (uint32_t i = 0; i < SPINS && !__all_sync(0xffffffffu, parked(smem_u32(&sm.done[0]), 0)); i++) {}
    } else if (warp == P::ISSUER_O) {
        // ---- O = w V
        constexpr uint32_t ID_O = idesc_of(KIND, 128, HD, 1);
        const uint64_t v_desc = umma_desc_of(smem_u32(sm.v[0]), KT * 128, 1024, 2);
        for (int i = 0, t0 = 0; more && !gave_up(); t0 += it.n_tiles, more = item_at(++i, it)) {
            for (int t = t0; t < t0 + it.n_tiles && !gave_up(); t++) {
                const int st = t % STAGES, ob = t % NO;
                wait(&sm.vready[st], (t / STAGES) & 1);
                if (t >= NO) wait(&sm.ofree[ob], (t / NO - 1) & 1);
                wait(&sm.pfull[t % NS], (t / NS) & 1);
                tc_fence_after();
                const uint32_t w = tmem + P::S0 + (t % NS) * P::SREG, d = tmem + P::O0 + ob * HD;
                const uint64_t b = v_desc + (uint32_t)(st * (P::TILE >> 4));
                if (elected()) {
#pragma unroll
                    for (int k = QP - 1; k >= 0; k--)
#pragma unroll
                        for (int ks = 0; ks < KT / 16; ks++)
                            // 16 keys of all dims: 64-dim halves KT * 128 bytes apart, groups of 8 keys 1024 bytes apart
                            mma_ts(d, w + (ks >> 1) * (QP * 16) + k * 16 + (ks & 1) * 8, b + (ks * 2048 >> 4), ID_O, k < QP - 1 || ks > 0);
                    tc_commit(smem_u32(&sm.ofull[ob]));
                    tc_commit(smem_u32(&sm.vfree[st]));
                }
                __syncwarp();
            }
        }
        if (elected()) tc_commit(smem_u32(&sm.done[1]));
        __syncwarp();
        for (uint32_t i = 0; i < SPINS && !__all_sync(0xffffffffu, parked(smem_u32(&sm.done[1]), 0)); i++) {}
    } else if (warp == P::LOOKER) {
        // ---- values that not every row sees
        for (int i = 0, t0 = 0; more && !gave_up(); t0 += it.n_tiles, more = item_at(++i, it))
        for (int j = 0; j < it.n_tiles && !gave_up(); j++) {
            const int st = (t0 + j) % STAGES, key0 = it.key(j), p_min = it.p_min(), p_max = it.p_max();
            wait(&sm.vfull[st], ((t0 + j) / STAGES) & 1);
            if (it.edge(a, key0)) {
                // a quarter of the warp per row of 128 bytes, so that neighbouring lanes read neighbouring pieces
                uint32_t odd[2] = {0, 0};
#pragma unroll 4
                for (int x = 0; x < KT / 4; x++) {
                    const int r = 4 * x + (lane >> 3), k = key0 + r;
                    const bool some = k <= p_max && (a.window <= 0 || k > p_min - a.window || k < a.first);
                    const bool every = k <= p_min && (a.window <= 0 || k > p_max - a.window || k < a.first);
                    bool bad = false;
                    if (some && !every) {
#pragma unroll
                        for (int h = 0; h < HD / 64; h++) {
                            const uint4 y = *(const uint4*)(sm.v[st] + h * (KT * 128) + r * 128 + (lane & 7) * 16);
                            const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                if (KIND == KIND_F16) bad = bad || (u[i] & 0x7c00u) == 0x7c00u || (u[i] & 0x7c000000u) == 0x7c000000u;
                                else bad = bad || (u[i] & 0x7f80u) == 0x7f80u || (u[i] & 0x7f800000u) == 0x7f800000u;
                            }
                        }
                    }
                    const uint32_t votes = __ballot_sync(0xffffffffu, bad);
                    const bool row_bad = votes >> (lane & 24) & 0xff;
                    if (row_bad || !some) {
#pragma unroll
                        for (int h = 0; h < HD / 64; h++) *(uint4*)(sm.v[st] + h * (KT * 128) + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    if (votes)
                        for (int i = 0; i < 4; i++)
                            if (votes >> (8 * i) & 0xff) odd[x >> 3] |= 1u << ((4 * x + i) & 31);
                }
                if (lane == 0) sm.odd[st] = odd[0] | (unsigned long long)odd[1] << 32;
                fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.vready[st]));
        }
    } else {
        const int w = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;      // half of the tile's keys, or of the dims; row of the 128
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        int odds = 0;
        bool again = false;
        for (int item = 0, t0 = 0; more; t0 += it.n_tiles, more = item_at(++item, it)) {
        if (it.n_tiles == 0) continue;
        const int n_tiles = it.n_tiles, row0 = it.row0, row1 = it.row1, kvh = it.kvh, s = it.s;
        const int row = row0 + r / a.group, h = kvh * a.group + r % a.group;
        const bool on = r < a.rq * a.group && row <= row1;
        const int p = on ? it.base + row : -1;
        // q's rows through shared memory (where odd weights will lie): read row by row, taken back a row a thread.  Piece c of row i
        // lies at c ^ i, so that neither side meets a bank twice.
        float4* const stage = reinterpret_cast<float4*>(sm.stage);
        float* const odd_w = sm.stage;
        constexpr int ROW4 = HD / 4, SHARE = 128 * ROW4 / 512;
        float qs = 1.0f;
        {
            float4 y[SHARE];
            const uint32_t inv = (65535 + a.group) / a.group;      // i / group = i inv / 2^16 below 128
#pragma unroll
            for (int u = 0; u < SHARE; u++) {
                const int x = u * 512 + tid, i = x / ROW4, ig = (int)(i * inv >> 16), ri = row0 + ig;
                y[u] = make_float4(0, 0, 0, 0);
                if (i < a.rq * a.group && ri <= row1 && 4 * (x % ROW4) < hd)
                    y[u] = *(const float4*)(a.q + ((size_t)s * a.rows + ri) * a.q_ld + (size_t)(kvh * a.group + i - ig * a.group) * hd + 4 * (x % ROW4));
            }
            if (again) asm volatile("bar.sync 2, 512;" ::: "memory");      // the item before has left shared memory
            again = true;
#pragma unroll
            for (int u = 0; u < SHARE; u++) {
                const int x = u * 512 + tid, i = x / ROW4;
                stage[i * ROW4 + ((x % ROW4) ^ (i & (ROW4 - 1)))] = y[u];
            }
        }
        asm volatile("bar.sync 2, 512;" ::: "memory");
        {
            // a quarter of a row a thread: scaled, split, into tensor memory part by part
            constexpr int QUARTER = HD / 4;
            const int qt = warp >> 2;
            const float sl = a.scale * LOG2E;
            float x[QUARTER], top = 0.0f;
#pragma unroll
            for (int d = 0; d < QUARTER; d += 4) {
                const float4 z = stage[r * ROW4 + ((qt * (QUARTER / 4) + d / 4) ^ (r & (ROW4 - 1)))];
                x[d] = z.x * sl; x[d + 1] = z.y * sl; x[d + 2] = z.z * sl; x[d + 3] = z.w * sl;
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(x[d + i]));
            }
            if (KIND == KIND_F16) {
                float* const tops = &sm.fin[0][0][0];              // [4][128]
                tops[qt * 128 + r] = top;
                asm volatile("bar.sync 2, 512;" ::: "memory");
                top = fmaxf(fmaxf(tops[r], tops[128 + r]), fmaxf(tops[256 + r], tops[384 + r]));
                // 2^e with top * 2^e in [2^13, 2^14)
                int ex = top > 0.0f && top < INFINITY ? 13 - (int)((__float_as_uint(top) >> 23) & 255) + 127 : 0;
                ex = max(-100, min(100, ex));
                const float f = __uint_as_float((uint32_t)(127 + ex) << 23);
#pragma unroll
                for (int d = 0; d < QUARTER; d++) x[d] *= f;
                qs = __uint_as_float((uint32_t)(127 - ex) << 23);
            }
#pragma unroll
            for (int k = 0; k < QP; k++) {
                uint32_t pk[QUARTER / 2];
#pragma unroll
                for (int i = 0; i < QUARTER / 2; i++) pk[i] = take_part<KIND>(x[2 * i], x[2 * i + 1]);
                const uint32_t at = tmem + lanes + P::Q0 + k * HALF + qt * (QUARTER / 2);
                if (HD == 128) tc_st16(at, pk);
                else tc_st8(at, pk);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.qfull));
        }
        auto sees = [&](int k) { return k <= p && (a.window <= 0 || k > p - a.window || k < a.first); };
        if (warp < P::OUT) {
            // ---- softmax
            float m = -INFINITY, l = 0.0f;                         // the denominator of this half's keys, relative to m
            for (int j = 0; j < n_tiles; j++) {
                const int t = t0 + j, b = t & 1, key0 = it.key(j) + 32 * w;
                wait(&sm.sfull[t % NS], (t / NS) & 1);
                tc_fence_after();
                const uint32_t at = tmem + lanes + P::S0 + (t % NS) * P::SREG;
                const bool edge = it.edge(a, it.key(j));
                float v[32];
                tm_ld<32>(at + P::LEAD + w * 32, v);
                if (edge) {
                    const int up = p - key0, dn = a.window > 0 ? p - a.window - key0 : -1, fi = a.window > 0 ? a.first - key0 : 0;
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = i <= up && (i > dn || i < fi) ? v[i] : -INFINITY;
                }
                float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int i = 4; i < 28; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; k++) top[k] = fmaxf(fmaxf(top[k], v[i + k]), v[i + 4 + k]);
#pragma unroll
                for (int k = 0; k < 4; k++) top[k] = fmaxf(top[k], v[28 + k]);
                const float tm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * qs;
                // the row's other half; behind the barrier both halves of S are in registers
                sm.top[b][w][r] = tm;
                tc_fence_before();
                asm volatile("bar.sync 3, 256;" ::: "memory");
                tc_fence_after();
                const float m_new = fmaxf(fmaxf(m, tm), sm.top[b][1 - w][r]), ms = m_new == -INFINITY ? 0.0f : m_new - SHIFT;
                const float c = m == -INFINITY ? 0.0f : pow2f(m - m_new);
                if (w == 0) sm.corr[t & 7][r] = c;
                m = m_new;
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 x = fma2(make_float2(v[i], v[i + 1]), make_float2(qs, qs), make_float2(-ms, -ms));
                    v[i] = pow2f(x.x);
                    v[i + 1] = pow2f(x.y);
                    sum[i >> 1 & 1] = add2(sum[i >> 1 & 1], make_float2(v[i], v[i + 1]));
                }
                l = fmaf(l, c, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
                unsigned long long odd = 0;
                if (edge) {
                    wait(&sm.vready[t % STAGES], (t / STAGES) & 1);
                    odd = __shfl_sync(0xffffffffu, sm.odd[t % STAGES], 0);
                    if (odd) {                                     // rare
                        if (odds > 0) wait(&sm.oddfree, (odds - 1) & 1);
                        odds++;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (odd >> (32 * w + i) & 1) odd_w[(32 * w + i) * 128 + r] = sees(key0 + i) ? v[i] : -1.0f;
                    }
                }
                if (tid == 0) sm.odd_of[t & 7] = odd;
#pragma unroll
                for (int k = 0; k < QP; k++) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) pk[i] = take_part<KIND>(v[2 * i], v[2 * i + 1]);
                    tc_st16(at + w * (QP * 16) + k * 16, pk);
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.pfull[t % NS]));
            }
            sm.fin[w][0][r] = l;
            sm.fin[w][1][r] = m;
            asm volatile("bar.sync 2, 512;" ::: "memory");
        } else {
            // ---- the running output: o = o corr + O
            float o[HALF];
#pragma unroll
            for (int d = 0; d < HALF; d++) o[d] = 0.0f;
            for (int j = 0; j < n_tiles; j++) {
                const int t = t0 + j, ob = t % NO;
                wait(&sm.ofull[ob], (t / NO) & 1);
                tc_fence_after();
                const float c = sm.corr[t & 7][r];
                const unsigned long long odd = __shfl_sync(0xffffffffu, sm.odd_of[t & 7], 0);
                constexpr int N = HD == 64 ? 32 : 16;
#pragma unroll
                for (int d0 = 0; d0 < HALF; d0 += N) {
                    float x[N];
                    tm_ld<N>(tmem + lanes + P::O0 + ob * HD + w * HALF + d0, x);
#pragma unroll
                    for (int d = 0; d < N; d += 2) {
                        const float2 y = fma2(make_float2(o[d0 + d], o[d0 + d + 1]), make_float2(c, c), make_float2(x[d], x[d + 1]));
                        o[d0 + d] = y.x;
                        o[d0 + d + 1] = y.y;
                    }
                }
                if (odd) {                                         // rare: values that are not finite, for the rows that see them
                    for (int i = 0; i < KT; i++) {
                        if (!(odd >> i & 1)) continue;
                        const float wt = odd_w[i * 128 + r];
                        if (wt < 0.0f) continue;
                        const int k = it.key(j) + i, pg = min(max(a.table[(size_t)s * a.max_pages + (k >> a.log_page)], 0), a.n_pages - 1);
                        const uint16_t* vr = (const uint16_t*)a.data + ((((size_t)2 * pg + 1) * a.n_kv + kvh) * a.page + (k & (a.page - 1))) * hd + w * HALF;
#pragma unroll
                        for (int d = 0; d < HALF; d++)
                            if (w * HALF + d < hd) o[d] = fmaf(wt, KIND == KIND_F16 ? fk_h2f(vr[d]) : __uint_as_float((uint32_t)vr[d] << 16), o[d]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sm.oddfree));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sm.ofree[ob]));
            }
            // the halves' denominators, the sink, the output
            asm volatile("bar.sync 2, 512;" ::: "memory");
            {
                const float m = sm.fin[0][1][r];
                float l = sm.fin[0][0][r] + sm.fin[1][0][r];
                if (a.sinks && on) l += m == -INFINITY ? 1.0f : pow2f(a.sinks[h] * LOG2E - m + SHIFT);
                const float inv = 1.0f / l;
                // through shared memory as q came, so that rows are written whole
#pragma unroll
                for (int d = 0; d < HALF; d += 4)
                    stage[r * ROW4 + ((w * (HALF / 4) + d / 4) ^ (r & (ROW4 - 1)))] = make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
                asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 4
                for (int x = tid - 32 * P::OUT; x < 128 * ROW4; x += 256) {
                    const int i = x / ROW4, ig = (int)(i * ((65535u + a.group) / a.group) >> 16), ri = row0 + ig;
                    if (i < a.rq * a.group && ri <= row1 && 4 * (x % ROW4) < hd)
                        *(float4*)(a.out + ((size_t)s * a.rows + ri) * a.n_heads * hd + (size_t)(kvh * a.group + i - ig * a.group) * hd + 4 * (x % ROW4)) =
                            stage[i * ROW4 + ((x % ROW4) ^ (i & (ROW4 - 1)))];
                }
            }
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == P::ISSUER_S) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int KIND, int HD> int launch_prompt(fk_ctx* ctx, cudaStream_t st, const PromptArgs& a, unsigned grid) {
    auto kern = attn_prompt_kernel<KIND, HD>;
    const size_t smem = sizeof(PromptSmem<KIND, HD>) + 1024;
    static thread_local bool ready[64] = {};
    if (!ready[ctx->device & 63]) {
        FK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), FK_KERNEL);
        FK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared), FK_KERNEL);
        ready[ctx->device & 63] = true;
    }
    FK_CUDA(launch(kern, dim3(grid), dim3(Plan<KIND, HD>::THREADS), smem, st, a), FK_LAUNCH);
    return FK_OK;
}

}  // namespace

// Whether this kernel takes the call, else attn_paged_kernel does.
bool fk_attn_prompt_takes(fk_ctx* ctx, const fk_pages* p, int rows, int n_heads) {
    const int group = n_heads / p->n_kv;
    if (p->kind == KIND_F32 || group > 128) return false;
    if ((long long)p->n_pages * 2 * p->n_kv * p->page > 0x7fffffffLL) return false;      // a token's row number is 32 bits
    // This kernel takes 19 ns an SM for a key of a tile of 128 columns, whatever of the tile is filled, and does not split the
    // keys; the other takes 13 ns an SM for a key of 16 columns and spreads over all SMs (bf16, heads of 128; f16 heads of 64: 15
    // and 7).  24/8 heads of 128, one sequence after 8000 tokens, us here / there: 64 rows 167 / 84, 128 rows 170 / 152, 256
    // rows 172 / 293; four sequences: 24 rows 167 / 133, 43 rows 169 / 224.  64/8 heads of 64, f16, 64 rows 119 / 107, 128 rows
    // 121 / 206.  f32 pages stay there, as 128 columns of three-part products have no kernel here: 512 rows of 24/8 heads of 128
    // into an empty cache 69 us, four of 900 rows after 8000 tokens 7.5 ms (bf16 here: 1.05).
    const long long tiles = (long long)p->n_seqs * p->n_kv * ((rows + 128 / group - 1) / (128 / group));
    const long long blocks = (long long)p->n_seqs * p->n_kv * (((long long)rows * group + 15) / 16);
    return 3 * blocks > 5 * ctx->sm_count * ((tiles + ctx->sm_count - 1) / ctx->sm_count);
}

int fk_attn_prompt_launch(fk_ctx* ctx, cudaStream_t st, const fk_pages* p, int layer, const float* q, int q_ld, int rows, const int* n_new, int n_heads,
                          float scale, int window, int first, const float* sinks, float* out) {
    PromptArgs a{};
    char* data = (char*)p->data_dev + (size_t)layer * page_bytes(p) * p->n_pages;
    const int rc = fk_make_map_2d(&a.map, 1, data, p->head_dim, (uint64_t)p->n_pages * 2 * p->n_kv * p->page, 64, p->page < KT ? p->page : KT, 3);
    if (rc != FK_OK) return rc;
    a.data = data;
    a.table = p->table_dev;
    a.lens = p->lens_dev;
    a.n_new = n_new;
    a.q = q;
    a.sinks = sinks;
    a.out = out;
    a.err = ctx->err_flag;
    a.scale = scale;
    a.q_ld = q_ld;
    a.rows = rows;
    a.n_seqs = p->n_seqs;
    a.n_heads = n_heads;
    a.n_kv = p->n_kv;
    a.group = n_heads / p->n_kv;
    a.head_dim = p->head_dim;
    a.page = p->page;
    a.log_page = p->page == 16 ? 4 : p->page == 32 ? 5 : p->page == 64 ? 6 : 7;
    a.n_pages = p->n_pages;
    a.max_pages = p->max_pages;
    a.window = window;
    a.first = first;
    a.rq = 128 / a.group;
    a.n_rb = (rows + a.rq - 1) / a.rq;
    const long long items = (long long)a.n_rb * a.n_seqs * a.n_kv, grid = items < ctx->sm_count ? items : ctx->sm_count;
    if (items > 0x7fffffffLL) return fk_fail(FK_UNSUPPORTED, "attention_paged: %d rows of %d sequences", rows, p->n_seqs);
    // shorter heads are zeros behind their last dim: the tiled copy fills what lies outside its tensor
    if (p->kind == KIND_F16) return p->head_dim <= 64 ? launch_prompt<KIND_F16, 64>(ctx, st, a, (unsigned)grid) : launch_prompt<KIND_F16, 128>(ctx, st, a, (unsigned)grid);
    return p->head_dim <= 64 ? launch_prompt<FK_BF16, 64>(ctx, st, a, (unsigned)grid) : launch_prompt<FK_BF16, 128>(ctx, st, a, (unsigned)grid);
}
