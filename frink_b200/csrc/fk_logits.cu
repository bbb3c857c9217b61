// Rules on logits: penalties for tokens that came before, biases, a grammar's mask, and the greedy pick, in one pass.
//
// Reads and writes 4 bytes a token of the vocabulary: bound by HBM where there are many rows, by one launch's latency
// where there is one.  A block takes a slice of a row: it counts the row's history inside the slice in shared memory (whole
// numbers, so the order of the atomics does not matter), then every logit is read, changed and written once, and the largest
// is kept as an order-preserving key that the block which arrives last for the row joins.
#include "fk_paged.cuh"

namespace {

constexpr int LR_THREADS = 256, LR_SLICE = 4096, LR_MAX_BLOCKS = 64, LR_ROWS = 64;

__device__ __forceinline__ unsigned long long key_of(float v, int i) {
    unsigned u = __float_as_uint(v != v ? -INFINITY : v);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned)(~i);
}
constexpr unsigned KEY_MINUS_INF = ~0xff800000u;

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
    int vocab, n_hist, slices;      // slices of LR_SLICE tokens a block walks
};

// The steps are rounded one by one, as written: no fused multiply-add.
__device__ __forceinline__ float penalised(float x, int c, float rep, float freq, float pres) {
    x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
    return __fsub_rn(__fsub_rn(x, __fmul_rn((float)c, freq)), pres);
}

__global__ void __launch_bounds__(LR_THREADS) rules_kernel(const RuleArgs a) {
    fk_paged::pdl_sync();
    __shared__ int count[LR_SLICE];
    __shared__ unsigned long long sk[LR_THREADS / 32];
    __shared__ bool last;
    const int row = blockIdx.y;
    const float* x = a.logits + (size_t)row * a.ld;
    const int* hist = a.history ? a.history + (size_t)row * a.n_hist : nullptr;
    const float* bias = a.bias ? a.bias + (size_t)row * a.bias_ld : nullptr;
    const unsigned* mask = a.mask ? (const unsigned*)a.mask + (size_t)row * a.mask_ld : nullptr;
    float* out = a.out + (size_t)row * a.vocab;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.history) { rep = a.penalties[3 * row]; freq = a.penalties[3 * row + 1]; pres = a.penalties[3 * row + 2]; }
    unsigned long long best = 0ull;
    for (int sl = 0; sl < a.slices; sl++) {
        const int lo = (blockIdx.x * a.slices + sl) * LR_SLICE, n = min(LR_SLICE, a.vocab - lo);
        if (n <= 0) break;
        if (hist) {
            for (int i = threadIdx.x; i < LR_SLICE; i += LR_THREADS) count[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < a.n_hist; i += LR_THREADS) {
                const int t = hist[i] - lo;
                if (t >= 0 && t < n && hist[i] >= 0) atomicAdd(&count[t], 1);
            }
            __syncthreads();
        }
        constexpr int U = 8;
        for (int i0 = threadIdx.x; i0 < n; i0 += U * LR_THREADS) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; u++) v[u] = i0 + u * LR_THREADS < n ? x[lo + i0 + u * LR_THREADS] : 0.0f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + u * LR_THREADS;
                if (i >= n) continue;
                float y = v[u];
                if (hist) {
                    const int c = count[i];
                    if (c > 0) y = penalised(y, c, rep, freq, pres);
                }
                if (bias) y = __fadd_rn(y, bias[lo + i]);
                if (mask && !((mask[(lo + i) >> 5] >> ((lo + i) & 31)) & 1u)) y = -INFINITY;
                out[lo + i] = y;
                best = max(best, key_of(y, lo + i));
            }
        }
        __syncthreads();
    }
    if (!a.tokens) return;
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
            a.tokens[row] = (unsigned)(b >> 32) == KEY_MINUS_INF ? -1 : (int)(~(unsigned)(b & 0xffffffffull));
            a.cnt[row] = 0;
        }
    }
}

}  // namespace

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
    if (out_dev == logits_dev && ld != (size_t)vocab) return fk_fail(FK_INVALID, "logit_rules: logits are changed in place only where their rows are packed");
    if (vocab > 0x7fffffff - LR_SLICE * LR_MAX_BLOCKS) return fk_fail(FK_UNSUPPORTED, "logit_rules: %d logits", vocab);
    FkDeviceGuard g(ctx->device);
    const int slices_all = (vocab + LR_SLICE - 1) / LR_SLICE, slices = (slices_all + LR_MAX_BLOCKS - 1) / LR_MAX_BLOCKS;
    const int blocks = (slices_all + slices - 1) / slices;
    for (int r0 = 0; r0 < n_rows; r0 += LR_ROWS) {          // the workspace holds the keys of LR_ROWS rows
        const int n = n_rows - r0 < LR_ROWS ? n_rows - r0 : LR_ROWS;
        RuleArgs a{logits_dev + (size_t)r0 * ld, ld, history_dev ? history_dev + (size_t)r0 * history : nullptr, penalties_dev ? penalties_dev + 3 * (size_t)r0 : nullptr,
                   bias_dev ? bias_dev + (size_t)r0 * bias_ld : nullptr, mask_dev ? mask_dev + (size_t)r0 * mask_ld : nullptr, bias_ld, mask_ld,
                   out_dev + (size_t)r0 * vocab, tokens_dev ? tokens_dev + r0 : nullptr, ctx->argmax_ws, ctx->argmax_cnt, vocab, history, slices};
        FK_CUDA(fk_paged::launch(rules_kernel, dim3(blocks, n), dim3(LR_THREADS), 0, (cudaStream_t)stream, a), FK_LAUNCH);
        FK_CUDA(cudaGetLastError(), FK_LAUNCH);
        ctx->launches++;
    }
    return FK_OK;
}
