// The pool of a paged KV cache: growing, forking, freeing and compacting sequences' pages, and the append of new keys and
// values (with their rotation) into them.
//
// Tables, lengths and reference counts live on the device and one block decides: every decision is a prefix sum (the k-th
// missing page of the call takes the k-th free page of the pool, counted from 0), so it depends on the state alone and not on
// the order in which threads arrive, and a step captured in a graph can grow its sequences by itself.  The bookkeeping reads
// 4 bytes a page and stops at the last page it needs; what costs is the copying of page data, bound by HBM.  One block's scan
// shows in large pools: a page more for each of 64 sequences behind 44800 used pages of 50000 takes 23 us (6 behind 1920 of
// 2048), compacting such a pool where nothing moves 37 us (9).
#include "fk_paged.cuh"

#include <cmath>

using namespace fk_paged;

namespace {

constexpr int BK = 1024;        // threads of the deciding block

struct SeqList {
    int n;
    int id[MAX_LIST];
};
struct ForkList {
    int n;
    int src[MAX_LIST], dst[MAX_LIST], len[MAX_LIST];
};
// what the copy kernels read: page numbers, and how many tokens of the page
struct CopyItem {
    int src, dst, part, pad;
};

// Whether at least `need` pages are free; the scan stops at the block of pages that holds the last of them.
__device__ bool enough_free(const int* __restrict__ refs, int n_pages, int need, int* part) {
    int found = 0, total;
    for (int p0 = 0; p0 < n_pages && found < need; p0 += 4 * BK) {
        int mine = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int p = p0 + 4 * threadIdx.x + u;
            mine += p < n_pages && refs[p] == 0;
        }
        block_prefix(mine, part, &total);
        found += total;
    }
    return found >= need;
}

// Calls take(k, page) for the lowest `need` free pages, k = 0, 1, ... in ascending order of page (each by one thread).
template <typename F> __device__ void take_free(const int* refs, int n_pages, int need, int* part, F take) {
    int found = 0, total;
    for (int p0 = 0; p0 < n_pages && found < need; p0 += 4 * BK) {
        int mine = 0;
        bool is[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int p = p0 + 4 * threadIdx.x + u;
            is[u] = p < n_pages && refs[p] == 0;
            mine += is[u];
        }
        int k = found + block_prefix(mine, part, &total);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (is[u] && k < need) take(k, p0 + 4 * (int)threadIdx.x + u);
            k += is[u];
        }
        found += total;
    }
}

// ---- grow: every sequence's missing pages are one run behind its last page; the prefix sum of the runs' lengths ranks them
__global__ void __launch_bounds__(BK)
grow_kernel(int* __restrict__ table, const int* __restrict__ lens, int* refs, int n_pages, int page, int n_seqs, int max_pages,
            const int* __restrict__ n_new_dev, int n_new, int* __restrict__ err) {
    pdl_sync();
    __shared__ int part[33];
    __shared__ int first[MAX_SEQS], off[MAX_SEQS + 1];
    __shared__ int bad;
    __shared__ unsigned long long all;               // missing pages in all: the tables together may claim more than 32 bits count
    if (threadIdx.x == 0) {
        bad = 0;
        all = 0;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int s = warp; s < n_seqs; s += BK / 32) {
        const int len = lens[s], add = n_new_dev ? n_new_dev[s] : n_new;
        const long long upto = (long long)len + add;
        int f = 0, want = 0;
        if (len < 0 || add < 0 || upto > (long long)max_pages * page) {
            if (lane == 0) bad = 1;
        } else if (add > 0) {
            want = (int)((upto + page - 1) / page);
            f = (len + page - 1) / page;
            for (; f < want; f += 32) {              // first entry without a page
                const bool none = f + lane < want && table[(size_t)s * max_pages + f + lane] < 0;
                const unsigned b = __ballot_sync(0xffffffffu, none);
                if (b) {
                    f += __ffs(b) - 1;
                    break;
                }
            }
            f = min(f, want);
        }
        if (lane == 0) {
            first[s] = f;
            off[s] = want - f;
            if (want > f) atomicAdd(&all, (unsigned long long)(want - f));
        }
    }
    __syncthreads();
    if (bad || all > (unsigned long long)n_pages) {
        if (threadIdx.x == 0) fk_raise(err, bad ? 95 : 96);
        return;
    }
    // exclusive prefix over the sequences, a run of them per thread
    constexpr int PER = MAX_SEQS / BK;
    int mine[PER], sum = 0, need;
#pragma unroll
    for (int u = 0; u < PER; u++) {
        const int s = threadIdx.x * PER + u;
        mine[u] = s < n_seqs ? off[s] : 0;
        sum += mine[u];
    }
    int at = block_prefix(sum, part, &need);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; u++) {
        const int s = threadIdx.x * PER + u;
        if (s < n_seqs) off[s] = at;
        at += mine[u];
    }
    if (threadIdx.x == 0) off[n_seqs] = need;
    __syncthreads();
    if (need == 0) return;
    if (!enough_free(refs, n_pages, need, part)) {
        if (threadIdx.x == 0) fk_raise(err, 96);
        return;
    }
    __syncthreads();
    take_free(refs, n_pages, need, part, [&](int k, int p) {
        int lo = 0, hi = n_seqs - 1;                 // the last sequence whose first missing page has rank <= k
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (off[mid] <= k) lo = mid; else hi = mid - 1;
        }
        table[(size_t)lo * max_pages + first[lo] + k - off[lo]] = p;
        refs[p] = 1;                                 // only this thread looks at this page
    });
}

__global__ void advance_kernel(int* __restrict__ lens, int n_seqs, const int* __restrict__ n_new_dev, int n_new) {
    pdl_sync();
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < n_seqs) lens[s] += n_new_dev ? n_new_dev[s] : n_new;
}

// What a step moves: a launch's latency.  With the tokens' join (fk_logits.cu) in place of eleven elementwise launches: the captured
// step of a decoder of two layers, four sequences under rules, 112 -> 93 us (without rules six, 102 -> 91).
__global__ void moves_kernel(const int* __restrict__ tokens, const int* __restrict__ live, int n, int* __restrict__ ids, int* __restrict__ moves) {
    pdl_sync();
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s >= n) return;
    const int t = tokens[s];
    ids[s] = max(t, 0);
    moves[s] = live[s] != 0 && t >= 0;
}

// ---- free: a block per sequence
__global__ void __launch_bounds__(256)
free_kernel(int* __restrict__ table, int* __restrict__ lens, int* __restrict__ refs, int n_pages, int max_pages, const SeqList list, int* __restrict__ err) {
    pdl_sync();
    const int s = list.id[blockIdx.x];
    for (int i = threadIdx.x; i < max_pages; i += blockDim.x) {
        const int p = table[(size_t)s * max_pages + i];
        if (p < 0) continue;
        table[(size_t)s * max_pages + i] = -1;
        if (p >= n_pages) fk_raise(err, 97);
        else atomicSub(&refs[p], 1);
    }
    if (threadIdx.x == 0) lens[s] = 0;
}

// ---- fork
__global__ void __launch_bounds__(BK)
fork_kernel(int* table, int* lens, int* refs, int n_pages, int page, int max_pages, const ForkList list, CopyItem* __restrict__ items, int* __restrict__ err) {
    pdl_sync();
    __shared__ int part[33];
    __shared__ int s_n[MAX_LIST], s_rank[MAX_LIST], s_page[MAX_LIST];
    __shared__ int wrong;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = threadIdx.x;
    if (i == 0) wrong = 0;
    __syncthreads();
    int has = 0;
    if (i < list.n) {
        const int held = lens[list.src[i]], n = list.len[i] < 0 ? held : list.len[i];
        if (n < 0 || n > held || held > max_pages * page || lens[list.dst[i]] != 0 || table[(size_t)list.dst[i] * max_pages] >= 0) wrong = 98;
        s_n[i] = n;
        has = n % page != 0;
    }
    __syncthreads();
    // every page that is taken over must be one of the pool's
    if (!wrong) {
        for (int k = warp; k < list.n; k += BK / 32) {
            const int cnt = (s_n[k] + page - 1) / page;
            for (int j = lane; j < cnt; j += 32) {
                const int p = table[(size_t)list.src[k] * max_pages + j];
                if (p < 0 || p >= n_pages) wrong = 97;
            }
        }
    }
    int need;
    const int rank = block_prefix(has, part, &need);
    if (i < list.n) s_rank[i] = has ? rank : -1;
    __syncthreads();
    if (!wrong && need > 0 && !enough_free(refs, n_pages, need, part) && i == 0) wrong = 96;
    __syncthreads();
    if (wrong) {
        if (i == 0) fk_raise(err, wrong);
        if (i < list.n) items[i] = CopyItem{0, 0, 0, 0};
        return;
    }
    if (need > 0) take_free(refs, n_pages, need, part, [&](int k, int p) { s_page[k] = p; });
    __syncthreads();
    for (int k = warp; k < list.n; k += BK / 32) {
        const int n = s_n[k], full = n / page;
        const int* from = table + (size_t)list.src[k] * max_pages;
        int* to = table + (size_t)list.dst[k] * max_pages;
        for (int j = lane; j < full; j += 32) {
            const int p = from[j];
            to[j] = p;
            atomicAdd(&refs[p], 1);
        }
        if (lane == 0) {
            CopyItem it{0, 0, 0, 0};
            if (s_rank[k] >= 0) {
                const int p = s_page[s_rank[k]];
                to[full] = p;
                refs[p] = 1;
                it = CopyItem{from[full], p, n % page, 0};
            }
            items[k] = it;
            lens[list.dst[k]] = n;
        }
    }
}

// Four forks of 1000 tokens in 28 layers, with the frees before and the growth behind them, are 14 us, all of it latency: four
// dependent launches, three of them a chain of table reads, the scan for free pages, the table's and the counts' writes.
// The last, partly filled pages: `part` tokens of every head, K and V, of every layer.  blockIdx.x: fork, blockIdx.y: layer.
__global__ void __launch_bounds__(256)
copy_parts_kernel(char* __restrict__ data, const CopyItem* __restrict__ items, size_t layer_bytes, size_t page_bytes, int heads2, int head_bytes, int row_bytes) {
    pdl_sync();
    const CopyItem it = items[blockIdx.x];
    if (it.part == 0) return;
    const int n16 = it.part * row_bytes / 16;                    // 16-byte pieces of one head
    char* base = data + (size_t)blockIdx.y * layer_bytes;
    const char* src = base + (size_t)it.src * page_bytes;
    char* dst = base + (size_t)it.dst * page_bytes;
    for (int k = threadIdx.x; k < heads2 * n16; k += blockDim.x) {
        const size_t at = (size_t)(k / n16) * head_bytes + (size_t)(k % n16) * 16;
        *(uint4*)(dst + at) = *(const uint4*)(src + at);
    }
}

// ---- compact: lists in the workspace: [0] moves, [1] pages in use; from 16 on free pages below U, then used pages from U on
__global__ void __launch_bounds__(BK)
compact_kernel(int* refs, int n_pages, int* __restrict__ lists, int* __restrict__ used_out) {
    pdl_sync();
    __shared__ int part[33];
    int mine = 0, U;
    for (int p = threadIdx.x; p < n_pages; p += BK) mine += refs[p] != 0;
    block_prefix(mine, part, &U);
    int* holes = lists + 16;
    int* movers = holes + n_pages;
    int* map = movers + n_pages;                                 // new number of every page from U on
    int nh = 0, nm = 0;
    for (int p0 = 0; p0 < n_pages; p0 += BK) {
        const int p = p0 + threadIdx.x;
        const bool used = p < n_pages && refs[p] != 0;
        const bool hole = p < U && !used, mover = p >= U && used;
        int total;
        // one prefix for both: a page is a hole or a mover, holes in the low half, movers in the high half
        const int pre = block_prefix((hole ? 1 : 0) | (mover ? 1 << 16 : 0), part, &total);
        if (hole) holes[nh + (pre & 0xffff)] = p;
        if (mover) movers[nm + (pre >> 16)] = p;
        else if (p >= U && p < n_pages) map[p] = p;
        nh += total & 0xffff;
        nm += total >> 16;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < nm; k += BK) {
        const int from = movers[k], to = holes[k];
        refs[to] = refs[from];
        refs[from] = 0;
        map[from] = to;
    }
    if (threadIdx.x == 0) {
        lists[0] = nm;
        lists[1] = U;
        *used_out = U;
    }
}

// blocks below `table_blocks` rewrite the tables, the others copy pages: piece i of (layer, move) pairs.  Bound by HBM: 500 moves
// of 64 KB in 28 layers 313 us with the deciding block = 5.9 TB/s.
__global__ void __launch_bounds__(256)
move_kernel(char* __restrict__ data, int* __restrict__ table, const int* __restrict__ lists, int n_pages, size_t layer_bytes, size_t page_bytes, int n_layers,
            size_t table_len, int table_blocks, int* __restrict__ err) {
    pdl_sync();
    const int moves = lists[0], U = lists[1];
    if (moves == 0) return;
    const int *holes = lists + 16, *movers = holes + n_pages, *map = movers + n_pages;
    if ((int)blockIdx.x < table_blocks) {
        for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < table_len; i += (size_t)table_blocks * blockDim.x) {
            const int p = table[i];
            if (p < U) continue;
            if (p >= n_pages) fk_raise(err, 97);
            else table[i] = map[p];
        }
        return;
    }
    const size_t pieces = page_bytes / 16;
    const int tasks = moves * n_layers, step = gridDim.x - table_blocks;
    for (int t = blockIdx.x - table_blocks; t < tasks; t += step) {
        const int l = t / moves, k = t % moves;
        const uint4* src = (const uint4*)(data + (size_t)l * layer_bytes + (size_t)movers[k] * page_bytes);
        uint4* dst = (uint4*)(data + (size_t)l * layer_bytes + (size_t)holes[k] * page_bytes);
        for (size_t i = threadIdx.x; i < pieces; i += 4 * 256) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) if (i + u * 256 < pieces) v[u] = src[i + u * 256];
#pragma unroll
            for (int u = 0; u < 4; u++) if (i + u * 256 < pieces) dst[i + u * 256] = v[u];
        }
    }
}

// ---- rotation and append.  A block takes one row: the rotation factors of its position once, in shared memory, for all
// heads; then a group of 16 lanes per head, a lane holding 8 of its values = 4 rotation pairs.
// The angle p * theta^(-2i/d) loses its fraction in 32 bits at far positions (p = 125000: 0.004 turns), so it is taken in
// 64 bits, in turns, reduced to (-1/2, 1/2], and only then rounded; sincospif sees an argument of full relative precision.
// Bound by HBM: it reads q, k, v once, writes q once and k, v once in the pages' type.  4096 rows of 32/4 heads of 128 with
// norms into f16 pages: 30 us = 5.3 TB/s (two or three heads of a group requested together: 35 and 37 us, registers); 8 rows of
// 24/8 heads 3.5 us, one launch's latency.
struct RopeArgs {
    const float *q, *k, *v, *q_norm, *k_norm;
    float* q_out;
    void* data;                     // the layer's pages
    const int *table, *lens, *n_new;
    int* err;
    int q_ld, k_ld, v_ld, rows, n_heads, n_kv, head_dim, page, n_pages, max_pages, neox;
    float eps;
    double log2_theta;
};

template <int KIND> __device__ __forceinline__ void store4(void* base, size_t at, float4 v) {
    if (KIND == KIND_F32) {
        *(float4*)((float*)base + at) = v;
    } else if (KIND == KIND_F16) {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *(uint2*)((uint16_t*)base + at) = make_uint2(*(const uint32_t*)&a, *(const uint32_t*)&b);
    } else {
        uint32_t a, b;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(a) : "f"(v.y), "f"(v.x));
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(b) : "f"(v.w), "f"(v.z));
        *(uint2*)((uint16_t*)base + at) = make_uint2(a, b);
    }
}

template <int KIND> __global__ void __launch_bounds__(256) rope_paged_kernel(const RopeArgs a) {
    pdl_sync();
    const int r = blockIdx.x, s = r / a.rows, i = r % a.rows, hd = a.head_dim, half = hd >> 1;
    const int n = a.n_new ? min(a.n_new[s], a.rows) : a.rows;
    if (i >= n) return;
    const int len = a.lens[s];
    if (len < 0 || (long long)len + n > (long long)a.max_pages * a.page) {
        if (threadIdx.x == 0) fk_raise(a.err, 95);
        return;
    }
    const int p = len + i;
    const int pg = a.table[(size_t)s * a.max_pages + p / a.page];
    const bool held = pg >= 0 && pg < a.n_pages;
    if (!held && threadIdx.x == 0) fk_raise(a.err, 97);
    __shared__ float2 cs[64];
    if (threadIdx.x < half) {
        const double turns = (double)p * (exp2(-2.0 * threadIdx.x / hd * a.log2_theta) * 0.15915494309189533577);
        float sn, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
        cs[threadIdx.x] = make_float2(c, sn);
    }
    __syncthreads();
    const int sub = threadIdx.x & 15, items = hd >> 3;
    const bool on = sub < items;
    // the lane's 8 values: 8 in a row (pairs of neighbours), or 4 of each half (pairs half a head apart)
    const int i0 = a.neox ? 4 * sub : 8 * sub, i1 = a.neox ? half + 4 * sub : 8 * sub + 4;
    const size_t in_page = (size_t)(p % a.page) * hd, head_elems = (size_t)a.page * hd;
    for (int h = threadIdx.x >> 4; h < a.n_heads + 2 * a.n_kv; h += blockDim.x >> 4) {
        const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
        const int kh = is_q ? h : (h - a.n_heads) % a.n_kv;
        const float* src = is_q ? a.q + (size_t)r * a.q_ld + (size_t)h * hd : (is_v ? a.v + (size_t)r * a.v_ld : a.k + (size_t)r * a.k_ld) + (size_t)kh * hd;
        float4 x = make_float4(0, 0, 0, 0), y = x;
        if (on) {
            x = *(const float4*)(src + i0);
            y = *(const float4*)(src + i1);
        }
        if (!is_v) {
            const float* nw = is_q ? a.q_norm : a.k_norm;
            if (nw) {
                float sq = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
                const unsigned lanes = 0xffffu << (threadIdx.x & 16);
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sq += __shfl_xor_sync(lanes, sq, o);
                const float sc = 1.0f / sqrtf(sq / (float)hd + a.eps);
                if (on) {
                    const float4 w = *(const float4*)(nw + i0), z = *(const float4*)(nw + i1);
                    x.x *= sc * w.x; x.y *= sc * w.y; x.z *= sc * w.z; x.w *= sc * w.w;
                    y.x *= sc * z.x; y.y *= sc * z.y; y.z *= sc * z.z; y.w *= sc * z.w;
                }
            }
            if (on) {
                const float2 c0 = cs[4 * sub], c1 = cs[4 * sub + 1], c2 = cs[4 * sub + 2], c3 = cs[4 * sub + 3];
                const float4 u = x, w = y;
                if (a.neox) {
                    x = make_float4(u.x * c0.x - w.x * c0.y, u.y * c1.x - w.y * c1.y, u.z * c2.x - w.z * c2.y, u.w * c3.x - w.w * c3.y);
                    y = make_float4(u.x * c0.y + w.x * c0.x, u.y * c1.y + w.y * c1.x, u.z * c2.y + w.z * c2.x, u.w * c3.y + w.w * c3.x);
                } else {
                    x = make_float4(u.x * c0.x - u.y * c0.y, u.x * c0.y + u.y * c0.x, u.z * c1.x - u.w * c1.y, u.z * c1.y + u.w * c1.x);
                    y = make_float4(w.x * c2.x - w.y * c2.y, w.x * c2.y + w.y * c2.x, w.z * c3.x - w.w * c3.y, w.z * c3.y + w.w * c3.x);
                }
            }
        }
        if (!on) continue;
        if (is_q) {
            float* o = a.q_out + ((size_t)r * a.n_heads + h) * hd;
            *(float4*)(o + i0) = x;
            *(float4*)(o + i1) = y;
        } else if (held) {
            const size_t at = ((size_t)(2 * (size_t)pg + (is_v ? 1 : 0)) * a.n_kv + kh) * head_elems + in_page;
            store4<KIND>(a.data, at + i0, x);
            store4<KIND>(a.data, at + i1, y);
        }
    }
}

int list_ok(const char* what, const int* ids, int m, int n_seqs) {
    if (!ids || m < 1 || m > MAX_LIST) return fk_fail(FK_INVALID, "%s: a list of %d sequences (1 to %d)", what, m, MAX_LIST);
    for (int i = 0; i < m; i++) {
        if (ids[i] < 0 || ids[i] >= n_seqs) return fk_fail(FK_INVALID, "%s: sequence %d of %d", what, ids[i], n_seqs);
        for (int j = 0; j < i; j++) if (ids[j] == ids[i]) return fk_fail(FK_INVALID, "%s: sequence %d is listed twice", what, ids[i]);
    }
    return FK_OK;
}

}  // namespace

#define FK_PAGED_LAUNCHED() do { FK_CUDA(cudaGetLastError(), FK_LAUNCH); ctx->launches++; } while (0)

FK_EXPORT size_t fk_pages_workspace(fk_ctx* ctx, int n_pages) {
    if (!ctx || n_pages < 1) return 0;
    const size_t attn = (size_t)2 * ATTN_CTAS_PER_SM * ctx->sm_count * ATTN_RECORD * sizeof(float);
    const size_t lists = (16 + (size_t)3 * n_pages) * sizeof(int);
    return (WS_COUNTERS + (attn > lists ? attn : lists) + 255) & ~(size_t)255;
}

FK_EXPORT int fk_pages_grow(fk_ctx* ctx, void* stream, const fk_pages* p, const int* n_new_dev, int n_new) {
    const int rc = check("pages_grow", ctx, p);
    if (rc != FK_OK) return rc;
    if (!n_new_dev && n_new < 0) return fk_fail(FK_INVALID, "pages_grow: %d tokens", n_new);
    FkDeviceGuard g(ctx->device);
    FK_CUDA(launch(grow_kernel, dim3(1), dim3(BK), 0, (cudaStream_t)stream, p->table_dev, (const int*)p->lens_dev, p->refs_dev, p->n_pages, p->page,
                   p->n_seqs, p->max_pages, n_new_dev, n_new, ctx->err_flag), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_pages_advance(fk_ctx* ctx, void* stream, const fk_pages* p, const int* n_new_dev, int n_new) {
    const int rc = check("pages_advance", ctx, p);
    if (rc != FK_OK) return rc;
    if (!n_new_dev && n_new < 0) return fk_fail(FK_INVALID, "pages_advance: %d tokens", n_new);
    FkDeviceGuard g(ctx->device);
    FK_CUDA(launch(advance_kernel, dim3((p->n_seqs + 255) / 256), dim3(256), 0, (cudaStream_t)stream, p->lens_dev, p->n_seqs, n_new_dev, n_new), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_pages_moves(fk_ctx* ctx, void* stream, const int* tokens_dev, const int* live_dev, int n, int* ids_dev, int* moves_dev) {
    if (!ctx || !tokens_dev || !live_dev || !ids_dev || !moves_dev) return fk_fail(FK_INVALID, "pages_moves: null argument");
    if (n < 1) return fk_fail(FK_INVALID, "pages_moves: %d sequences", n);
    FkDeviceGuard g(ctx->device);
    FK_CUDA(launch(moves_kernel, dim3((n + 255) / 256), dim3(256), 0, (cudaStream_t)stream, tokens_dev, live_dev, n, ids_dev, moves_dev), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_pages_free(fk_ctx* ctx, void* stream, const fk_pages* p, const int* seqs_host, int m) {
    int rc = check("pages_free", ctx, p);
    if (rc == FK_OK) rc = list_ok("pages_free", seqs_host, m, p->n_seqs);
    if (rc != FK_OK) return rc;
    SeqList list;
    list.n = m;
    for (int i = 0; i < m; i++) list.id[i] = seqs_host[i];
    FkDeviceGuard g(ctx->device);
    FK_CUDA(launch(free_kernel, dim3(m), dim3(256), 0, (cudaStream_t)stream, p->table_dev, p->lens_dev, p->refs_dev, p->n_pages, p->max_pages, list,
                   ctx->err_flag), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_pages_fork(fk_ctx* ctx, void* stream, const fk_pages* p, const int* src_host, const int* dst_host, const int* n_host, int m) {
    int rc = check("pages_fork", ctx, p);
    if (rc == FK_OK) rc = list_ok("pages_fork: destinations", dst_host, m, p->n_seqs);
    if (rc != FK_OK) return rc;
    if (!src_host) return fk_fail(FK_INVALID, "pages_fork: null argument");
    if (p->n_layers > 65535) return fk_fail(FK_UNSUPPORTED, "pages_fork: %d layers", p->n_layers);
    ForkList list;
    list.n = m;
    for (int i = 0; i < m; i++) {
        if (src_host[i] < 0 || src_host[i] >= p->n_seqs) return fk_fail(FK_INVALID, "pages_fork: source %d of %d", src_host[i], p->n_seqs);
        for (int j = 0; j < m; j++)
            if (src_host[i] == dst_host[j]) return fk_fail(FK_INVALID, "pages_fork: sequence %d is a source and a destination", src_host[i]);
        list.src[i] = src_host[i];
        list.dst[i] = dst_host[i];
        list.len[i] = n_host ? n_host[i] : -1;
    }
    FkDeviceGuard g(ctx->device);
    CopyItem* items = (CopyItem*)((char*)p->ws_dev + WS_COUNTERS);
    FK_CUDA(launch(fork_kernel, dim3(1), dim3(BK), 0, (cudaStream_t)stream, p->table_dev, p->lens_dev, p->refs_dev, p->n_pages, p->page, p->max_pages, list,
                   items, ctx->err_flag), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    const int row = p->head_dim * elem_bytes(p->kind);
    FK_CUDA(launch(copy_parts_kernel, dim3(m, p->n_layers), dim3(256), 0, (cudaStream_t)stream, (char*)p->data_dev, (const CopyItem*)items,
                   page_bytes(p) * p->n_pages, page_bytes(p), 2 * p->n_kv, p->page * row, row), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_pages_compact(fk_ctx* ctx, void* stream, const fk_pages* p, int* used_dev) {
    const int rc = check("pages_compact", ctx, p);
    if (rc != FK_OK) return rc;
    if (!used_dev) return fk_fail(FK_INVALID, "pages_compact: null argument");
    if ((long long)p->n_layers * p->n_pages > 0x7fffffffLL) return fk_fail(FK_UNSUPPORTED, "pages_compact: %d layers of %d pages", p->n_layers, p->n_pages);
    FkDeviceGuard g(ctx->device);
    int* lists = (int*)((char*)p->ws_dev + WS_COUNTERS);
    FK_CUDA(launch(compact_kernel, dim3(1), dim3(BK), 0, (cudaStream_t)stream, p->refs_dev, p->n_pages, lists, used_dev), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    const size_t table_len = (size_t)p->n_seqs * p->max_pages;
    const int table_blocks = (int)((table_len + 4095) / 4096 > 64 ? 64 : (table_len + 4095) / 4096);
    FK_CUDA(launch(move_kernel, dim3(table_blocks + 8 * ctx->sm_count), dim3(256), 0, (cudaStream_t)stream, (char*)p->data_dev, p->table_dev, (const int*)lists,
                   p->n_pages, page_bytes(p) * p->n_pages, page_bytes(p), p->n_layers, table_len, table_blocks, ctx->err_flag), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}

FK_EXPORT int fk_rope_kv_paged(fk_ctx* ctx, void* stream, const fk_pages* p, int layer, const float* q_dev, const float* k_dev, const float* v_dev, int q_ld,
                               int k_ld, int v_ld, int rows, const int* n_new_dev, int n_heads, float theta, int neox, const float* q_norm_dev,
                               const float* k_norm_dev, float norm_eps, float* q_out_dev) {
    const int rc = check("rope_kv_paged", ctx, p, layer);
    if (rc != FK_OK) return rc;
    if (!q_dev || !k_dev || !v_dev || !q_out_dev) return fk_fail(FK_INVALID, "rope_kv_paged: null argument");
    if (rows < 1 || n_heads < 1 || n_heads > 65535 || (long long)rows * p->n_seqs > 0x7fffffffLL) return fk_fail(FK_INVALID, "rope_kv_paged: %d rows, %d heads", rows, n_heads);
    if (!(theta > 0.0f) || std::isinf(theta)) return fk_fail(FK_INVALID, "rope_kv_paged: theta %g", (double)theta);
    if ((q_norm_dev == nullptr) != (k_norm_dev == nullptr)) return fk_fail(FK_INVALID, "rope_kv_paged: q and k norm weights come together");
    if ((((uintptr_t)q_dev | (uintptr_t)k_dev | (uintptr_t)v_dev | (uintptr_t)q_out_dev | (uintptr_t)q_norm_dev | (uintptr_t)k_norm_dev) & 15) || (q_ld & 3) ||
        (k_ld & 3) || (v_ld & 3) || q_ld < n_heads * p->head_dim || k_ld < p->n_kv * p->head_dim || v_ld < p->n_kv * p->head_dim)
        return fk_fail(FK_INVALID, "rope_kv_paged: inputs must be 16-byte aligned, row strides multiples of 4 and at least a row");
    if (q_out_dev == q_dev && q_ld != n_heads * p->head_dim) return fk_fail(FK_INVALID, "rope_kv_paged: q is rotated in place only where its rows are packed");
    FkDeviceGuard g(ctx->device);
    RopeArgs a{q_dev, k_dev, v_dev, q_norm_dev, k_norm_dev, q_out_dev, (char*)p->data_dev + (size_t)layer * page_bytes(p) * p->n_pages, p->table_dev, p->lens_dev,
               n_new_dev, ctx->err_flag, q_ld, k_ld, v_ld, rows, n_heads, p->n_kv, p->head_dim, p->page, p->n_pages, p->max_pages, neox, norm_eps, log2((double)theta)};
    auto kern = p->kind == KIND_F32 ? rope_paged_kernel<KIND_F32> : p->kind == KIND_F16 ? rope_paged_kernel<KIND_F16> : rope_paged_kernel<FK_BF16>;
    FK_CUDA(launch(kern, dim3(rows * p->n_seqs), dim3(256), 0, (cudaStream_t)stream, a), FK_LAUNCH);
    FK_PAGED_LAUNCHED();
    return FK_OK;
}
