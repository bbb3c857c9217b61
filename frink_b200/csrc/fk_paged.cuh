// What the paged-cache kernels share: the pool's geometry, its argument checks, launches with programmatic serialization.
#pragma once
#include "fk_common.cuh"

// attention of many rows on the tensor cores' tcgen05 form (fk_attn_prompt.cu)
bool fk_attn_prompt_takes(fk_ctx* ctx, const fk_pages* p, int rows, int n_heads);
int fk_attn_prompt_launch(fk_ctx* ctx, cudaStream_t st, const fk_pages* p, int layer, const float* q, int q_ld, int rows, const int* n_new, int n_heads,
                          float scale, int window, int first, const float* sinks, float* out);

namespace fk_paged {

constexpr int MAX_SEQS = 4096, MAX_LIST = 64;
// workspace: arrival counters of the split attention (zero between calls), then scratch
constexpr size_t WS_COUNTERS = 8192;

constexpr int KIND_F32 = 0, KIND_F16 = 1;
static inline int elem_bytes(int kind) { return kind == KIND_F32 ? 4 : 2; }

// Null, range and alignment checks that every call on a pool makes; FK_OK or the failing call's status.
static inline int check(const char* what, fk_ctx* ctx, const fk_pages* p, int layer = 0) {
    if (!ctx || !p || !p->data_dev || !p->table_dev || !p->lens_dev || !p->refs_dev || !p->ws_dev) return fk_fail(FK_INVALID, "%s: null argument", what);
    if (p->kind != KIND_F32 && p->kind != KIND_F16 && p->kind != FK_BF16) return fk_fail(FK_UNSUPPORTED, "%s: pages of kind %d", what, p->kind);
    if (p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128) return fk_fail(FK_UNSUPPORTED, "%s: pages of %d tokens", what, p->page);
    if (p->head_dim < 8 || p->head_dim > 128 || (p->head_dim & 7)) return fk_fail(FK_UNSUPPORTED, "%s: heads of %d", what, p->head_dim);
    if (p->n_layers < 1 || p->n_pages < 1 || p->n_kv < 1 || p->n_kv > 1024 || p->max_pages < 1) return fk_fail(FK_INVALID, "%s: bad pool shape", what);
    if (p->n_seqs < 1 || p->n_seqs > MAX_SEQS) return fk_fail(FK_UNSUPPORTED, "%s: %d sequences", what, p->n_seqs);
    if ((long long)p->max_pages * p->page > 0x7fffffffLL - 1024) return fk_fail(FK_UNSUPPORTED, "%s: %d pages of %d tokens a sequence", what, p->max_pages, p->page);
    if (((uintptr_t)p->data_dev & 15) || ((uintptr_t)p->ws_dev & 255)) return fk_fail(FK_INVALID, "%s: pages must be 16-byte, the workspace 256-byte aligned", what);
    if (p->ws_bytes < fk_pages_workspace(ctx, p->n_pages)) return fk_fail(FK_INVALID, "%s: a workspace of %zu bytes", what, p->ws_bytes);
    if (layer < 0 || layer >= p->n_layers) return fk_fail(FK_INVALID, "%s: layer %d of %d", what, layer, p->n_layers);
    return FK_OK;
}

// bytes of one page of one layer
static inline size_t page_bytes(const fk_pages* p) { return (size_t)2 * p->n_kv * p->page * p->head_dim * elem_bytes(p->kind); }

// CTAs of the split attention's grid at most, per SM
constexpr int ATTN_CTAS_PER_SM = 4;
// one record: up to 16 query columns, each 128 sums, its maximum and its denominator
constexpr size_t ATTN_RECORD = (size_t)16 * 130;

#ifdef __CUDACC__
// The kernel may be scheduled while its predecessor in the stream still runs; it touches no memory before this.
__device__ __forceinline__ void pdl_sync() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// Exclusive prefix sum of one int a thread over a block of 1024 threads; *total for all.  `part` holds 33 ints.
__device__ __forceinline__ int block_prefix(int v, int* part, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int p = lane < nw ? part[lane] : 0, q = p;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, q, o);
            if (lane >= o) q += y;
        }
        part[lane] = q - p;
        if (lane == 31) part[32] = q;
    }
    __syncthreads();
    *total = part[32];
    return part[warp] + x - v;
}
#endif

}  // namespace fk_paged
