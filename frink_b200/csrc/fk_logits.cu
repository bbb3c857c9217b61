// Rules on logits: penalties for tokens that came before, biases, a grammar's mask, and the greedy pick, in one pass.
//
// Reads and writes 4 bytes a token of the vocabulary: bound by HBM where there are many rows, by one launch's latency
// where there is one.  A block takes a range of a row and first counts the row's history inside the range in shared memory, 16
// bits a token (whole numbers, so the order of the atomics does not matter): once per block, as many blocks as the SMs hold at a
// time, so that nothing but the stream of logits is left after it -- the next step's logits, bias and mask bits are requested
// before a step is worked on.  Every logit is read, changed and written once, and the largest is kept as an order-preserving key
// that the block which arrives last for the row joins.
// 64 x 201088 with bias, mask and a history of 1000, B200: blocks of 4096 logits that each read the history 52.8 us, with the
// loads ahead of it 36.5 us; this form 26.6 us = 4.0 TB/s, what is left is the latency of 40 KB in flight an SM: loads go to
// registers, since the counts (16 bits a token, 45 KB a block) hold the shared memory that a ring of copies would need.
#include "fk_paged.cuh"

namespace {

constexpr int LR_THREADS = 256, LR_PER_SM = 4, LR_MAX_BLOCKS = 64, LR_ROWS = 64;      // the workspace holds keys of 64 blocks of 64 rows
constexpr int LR_RANGE = 24480;                 // tokens of a block at most: their counts and the block's other shared memory are 48 KB
constexpr int LR_HISTORY = 65535;               // a count's 16 bits

// A key whose order is that of the values, then of descending index; 0 stands for no value.
__device__ __forceinline__ unsigned long long key_of(float v, int i) {
    unsigned u = v == 0.0f ? 0u : __float_as_uint(v);              // zeros of both signs are equal
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned)(~i);
}

struct RuleArgs {
    const float* logits;
    size_t ld;
    const int* history;
    const float *penalties, *bias;
    const int* mask;
    size_t bias_ld, mask_ld;
    float* out;
    int* tokens;
    unsigned long long* ws;
    unsigned* cnt;
    int vocab, n_hist, range;       // tokens of a block
};

// The steps are rounded one by one, as written: no fused multiply-add.
__device__ __forceinline__ float penalised(float x, int c, float rep, float freq, float pres) {
    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    return __fsub_rn(__fsub_rn(x, __fmul_rn((float)c, freq)), pres);
}

// VEC: rows are multiples of four on 16-byte boundaries, a thread takes four logits at a time.
template <bool VEC> __global__ void __launch_bounds__(LR_THREADS, LR_PER_SM) rules_kernel(const RuleArgs a) {
    fk_paged::pdl_sync();
    extern __shared__ __align__(16) unsigned count[];              // two counts a word
    __shared__ unsigned long long sk[LR_THREADS / 32];
    __shared__ bool last;
    const int row = blockIdx.y, lo = blockIdx.x * a.range, n = min(a.range, a.vocab - lo);
    const float* x = a.logits + (size_t)row * a.ld + lo;
    const float* bias = a.bias ? a.bias + (size_t)row * a.bias_ld + lo : nullptr;
    const unsigned* mask = a.mask ? (const unsigned*)a.mask + (size_t)row * a.mask_ld : nullptr;
    float* out = a.out + (size_t)row * a.vocab + lo;
    float top = -INFINITY;                                         // the largest so far; a thread's logits come in ascending order,
    int at = -1;                                                   // so the first of equal ones stays, and NaN never wins
    constexpr int W = VEC ? 4 : 1, U = VEC ? 2 : 8, E = U * W, STEP = LR_THREADS * W;      // logits together; groups, logits of a step
    struct Step {
        float v[E], b[E];
        unsigned bits[U];
    };
    const int first = threadIdx.x * W;
    auto request = [&](Step& s, int i0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * STEP;
            if (i < n) {
                if (VEC) *(float4*)(s.v + u * W) = *(const float4*)(x + i);
                else s.v[u] = x[i];
                if (bias) {
                    if (VEC) *(float4*)(s.b + u * W) = *(const float4*)(bias + i);
                    else s.b[u] = bias[i];
                }
                if (mask) s.bits[u] = mask[(lo + i) >> 5] >> ((lo + i) & 31);
            }
        }
    };
    Step cur;
    request(cur, first);
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    const bool counted = a.history != nullptr;
    if (counted) {
        const int* hist = a.history + (size_t)row * a.n_hist;
        rep = a.penalties[3 * row];
        freq = a.penalties[3 * row + 1];
        pres = a.penalties[3 * row + 2];
        for (int i = threadIdx.x; i < (n + 7) / 8; i += LR_THREADS) ((uint4*)count)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < a.n_hist; i += LR_THREADS) {
            const int id = hist[i], t = id - lo;                   // entries outside the vocabulary are empty places
            if (id >= 0 && t >= 0 && t < n) atomicAdd(&count[t >> 1], 1u << (16 * (t & 1)));
        }
        __syncthreads();
    }
    for (int i0 = first; i0 < n; i0 += U * STEP) {
        Step next;
        request(next, i0 + U * STEP);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * STEP;
            if (i >= n) break;
            float* v = cur.v + u * W;
            if (counted) {
                unsigned c[(W + 1) / 2];
                if (VEC) *(uint2*)c = *(const uint2*)(count + (i >> 1));
                else c[0] = count[i >> 1] >> (16 * (i & 1)) & 0xffffu;
                unsigned any = c[0];
                if (VEC) any |= c[(W - 1) / 2];
                if (any) {
#pragma unroll
                    for (int k = 0; k < W; k++) {
                        const int ck = (int)(c[k >> 1] >> (16 * (k & 1)) & 0xffffu);
                        if (ck > 0) v[k] = penalised(v[k], ck, rep, freq, pres);
                    }
                }
            }
            if (bias) {
#pragma unroll
                for (int k = 0; k < W; k++) v[k] = __fadd_rn(v[k], cur.b[u * W + k]);
            }
            if (mask) {
#pragma unroll
                for (int k = 0; k < W; k++) v[k] = cur.bits[u] >> k & 1u ? v[k] : -INFINITY;
            }
            if (VEC) *(float4*)(out + i) = make_float4(v[0], v[W - 3], v[W - 2], v[W - 1]);
            else out[i] = v[0];
            float most = v[0];
#pragma unroll
            for (int k = 1; k < W; k++) most = fmaxf(most, v[k]);
            if (most > top) {
#pragma unroll
                for (int k = W - 1; k >= 0; k--) if (v[k] == most) at = lo + i + k;
                top = most;
            }
        }
        cur = next;
    }
    if (!a.tokens) return;
    unsigned long long best = at < 0 ? 0ull : key_of(top, at);
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((threadIdx.x & 31) == 0) sk[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < LR_THREADS / 32; i++) best = max(best, sk[i]);
        a.ws[row * LR_MAX_BLOCKS + blockIdx.x] = best;
        __threadfence();
        last = atomicAdd(&a.cnt[row], 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (last && threadIdx.x < 32) {
        __threadfence();
        unsigned long long b = 0ull;
        for (int i = threadIdx.x; i < (int)gridDim.x; i += 32) b = max(b, ((volatile unsigned long long*)a.ws)[row * LR_MAX_BLOCKS + i]);
        for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        if (threadIdx.x == 0) {
            a.tokens[row] = b == 0ull ? -1 : (int)(~(unsigned)(b & 0xffffffffull));
            a.cnt[row] = 0;
        }
    }
}

// The picked tokens into their histories, a thread a sequence: a launch's latency.
__global__ void join_kernel(int* __restrict__ tokens, const int* __restrict__ moves, int n, int* __restrict__ history, int n_hist, int64_t* __restrict__ at) {
    fk_paged::pdl_sync();
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s >= n) return;
    int t = tokens[s];
    if (moves && moves[s] == 0) tokens[s] = t = -1;
    if (!history || t < 0) return;
    const int64_t a = at[s];
    history[(size_t)s * n_hist + (size_t)((uint64_t)a % (unsigned)n_hist)] = t;
    at[s] = a + 1;
}

}  // namespace

FK_EXPORT int fk_tokens_join(fk_ctx* ctx, void* stream, int* tokens_dev, const int* moves_dev, int n, int* history_dev, int history, int64_t* at_dev) {
    if (!ctx || !tokens_dev) return fk_fail(FK_INVALID, "tokens_join: null argument");
    if (n < 1) return fk_fail(FK_INVALID, "tokens_join: %d tokens", n);
    if (history_dev && (!at_dev || history < 1)) return fk_fail(FK_INVALID, "tokens_join: a history of %d tokens without their number", history);
    FkDeviceGuard g(ctx->device);
    FK_CUDA(fk_paged::launch(join_kernel, dim3((n + 255) / 256), dim3(256), 0, (cudaStream_t)stream, tokens_dev, moves_dev, n, history_dev, history, at_dev), FK_LAUNCH);
    FK_CUDA(cudaGetLastError(), FK_LAUNCH);
    ctx->launches++;
    return FK_OK;
}

FK_EXPORT int fk_logit_rules(fk_ctx* ctx, void* stream, const float* logits_dev, size_t ld, int n_rows, int vocab, const int* history_dev, int history,
                             const float* penalties_dev, const float* bias_dev, size_t bias_ld, const int* mask_dev, size_t mask_ld, float* out_dev,
                             int* tokens_dev) {
    if (!ctx || !logits_dev || !out_dev || n_rows < 1 || vocab < 1 || history < 0) return fk_fail(FK_INVALID, "logit_rules: bad argument");
    if (ld < (size_t)vocab) return fk_fail(FK_INVALID, "logit_rules: rows of %d logits, %zu apart", vocab, ld);
    if (history == 0) history_dev = nullptr;
    if (history > 0 && !history_dev) return fk_fail(FK_INVALID, "logit_rules: null history");
    if (history_dev && !penalties_dev) return fk_fail(FK_INVALID, "logit_rules: a history without penalties");
    if (bias_dev && bias_ld != 0 && bias_ld < (size_t)vocab) return fk_fail(FK_INVALID, "logit_rules: bias rows %zu apart", bias_ld);
    if (mask_dev && mask_ld != 0 && mask_ld < (size_t)(vocab + 31) / 32) return fk_fail(FK_INVALID, "logit_rules: mask rows of %zu words", mask_ld);
    if (n_rows == 1) ld = vocab;                             // no next row: how far it would be says nothing
    if (out_dev == logits_dev && ld != (size_t)vocab) return fk_fail(FK_INVALID, "logit_rules: logits are changed in place only where their rows are packed");
    if (history > LR_HISTORY) return fk_fail(FK_UNSUPPORTED, "logit_rules: a history of %d (at most %d)", history, LR_HISTORY);
    FkDeviceGuard g(ctx->device);
    const int rows_at_once = n_rows < LR_ROWS ? n_rows : LR_ROWS;
    // as many blocks a row as fill the SMs once, but no block below 2048 tokens or above its counts; ranges in whole mask words
    const int want = LR_PER_SM * ctx->sm_count / rows_at_once, most = (vocab + 2047) / 2048, least = (vocab + LR_RANGE - 1) / LR_RANGE;
    int blocks = want > most ? most : want;
    blocks = blocks < least ? least : blocks;
    if (blocks > LR_MAX_BLOCKS) blocks = LR_MAX_BLOCKS;
    const int range = ((vocab + blocks - 1) / blocks + 31) & ~31;
    if (range > LR_RANGE) return fk_fail(FK_UNSUPPORTED, "logit_rules: %d logits", vocab);
    blocks = (vocab + range - 1) / range;
    const uintptr_t bits = (uintptr_t)logits_dev | (uintptr_t)out_dev | (uintptr_t)bias_dev | (4 * (uintptr_t)ld) | (4 * (uintptr_t)vocab) | (4 * (uintptr_t)bias_ld);
    auto kern = bits & 15 ? rules_kernel<false> : rules_kernel<true>;
    for (int r0 = 0; r0 < n_rows; r0 += LR_ROWS) {          // the workspace holds the keys of LR_ROWS rows
        const int n = n_rows - r0 < LR_ROWS ? n_rows - r0 : LR_ROWS;
        RuleArgs a{logits_dev + (size_t)r0 * ld, ld, history_dev ? history_dev + (size_t)r0 * history : nullptr, penalties_dev ? penalties_dev + 3 * (size_t)r0 : nullptr,
                   bias_dev ? bias_dev + (size_t)r0 * bias_ld : nullptr, mask_dev ? mask_dev + (size_t)r0 * mask_ld : nullptr, bias_ld, mask_ld,
                   out_dev + (size_t)r0 * vocab, tokens_dev ? tokens_dev + r0 : nullptr, ctx->argmax_ws, ctx->argmax_cnt, vocab, history, range};
        FK_CUDA(fk_paged::launch(kern, dim3(blocks, n), dim3(LR_THREADS), history_dev ? 2 * (size_t)range + 16 : 0, (cudaStream_t)stream, a), FK_LAUNCH);
        FK_CUDA(cudaGetLastError(), FK_LAUNCH);
        ctx->launches++;
    }
    return FK_OK;
}
