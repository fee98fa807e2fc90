// The paged key-value cache: its writes (append) and its eviction by gathered attention weight.
//
// The reference leaves the cache itself to its caller; its get_block_table
// (src/unum_ops/sparse_kernel_extension/get_table_torch.py:29-44) only reads the table that maps a
// sequence's positions to physical tokens.  Position p of sequence b lives at token
//     table[b, p / P] * P + p % P            (P = page size, a power of two; 1 = the table get_block_table reads)
// of caches [n_tokens, Hk, D].
//
// append: token t of a batch is position token_pos_in_bs[t] - 1 of sequence token_to_bs[t] and its key and value
//   rows go to that position's token.  A copy: bound by HBM, 4 * Hk * D * 2 bytes a token.
//
// evict: of each sequence's pages in use the first `init`, the last `local` and the heaviest others stay, `budget`
//   in all.  A page's weight is the sum over kv heads and the page's positions of the weights that paged attention
//   gathered, taken in 64 bits and rounded to 32 once, so that no order of summation decides which page stays; ties
//   go to the lower index and a NaN ranks below every number.  The row closes up over what is evicted.
#include <cuda_runtime.h>

#include "common.cuh"

namespace {

// ------------------------------------------------------------------------------------------------ append
// One thread moves the same 16 bytes of the key and of the value row.  The rows' loads do not wait for the
// table's, and 2048 threads an SM keep 64 KB in flight, which covers HBM's latency.
struct AppendParams {
    const uint8_t *k, *v;
    uint8_t *kc, *vc;
    int64_t k_st, k_sh, v_st, v_sh, kc_st, kc_sh, vc_st, vc_sh;  // bytes
    const int32_t *table, *bs, *pos;
    int64_t bt_stride, n_pages, n_tokens, T, B;
    int32_t shift, chunks, hchunks_shift;  // 16-byte pieces of a token's row over all heads; log2 of one head's
};

__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = i / p.chunks;
    if (t >= p.T) return;
    const int32_t c = (int32_t)(i - t * p.chunks);
    const int64_t h = c >> p.hchunks_shift, o = (int64_t)(c & ((1 << p.hchunks_shift) - 1)) * 16;
    const int4 kv = __ldcs(reinterpret_cast<const int4 *>(p.k + t * p.k_st + h * p.k_sh + o));
    const int4 vv = __ldcs(reinterpret_cast<const int4 *>(p.v + t * p.v_st + h * p.v_sh + o));
    const int64_t b = __ldg(p.bs + t), at = (int64_t)__ldg(p.pos + t) - 1;
    if (b < 0 || b >= p.B || at < 0 || (at >> p.shift) >= p.n_pages) return;
    const int64_t page = __ldg(p.table + b * p.bt_stride + (at >> p.shift));
    const int64_t token = (page << p.shift) + (at & ((1 << p.shift) - 1));
    if (page < 0 || token >= p.n_tokens) return;
    *reinterpret_cast<int4 *>(p.kc + token * p.kc_st + h * p.kc_sh + o) = kv;
    *reinterpret_cast<int4 *>(p.vc + token * p.vc_st + h * p.vc_sh + o) = vv;
}

// ------------------------------------------------------------------------------------------------ evict
// One cluster of C blocks for each sequence; block r has a contiguous slice of its pages in use, with one 32-bit key
// a page in shared memory (the float's bits in an order that compares as unsigned; 0 = NaN).
//   keys     the sums, and the histogram of the keys' top digit;
//   select   radix selection over four 8-bit digits: every block adds up the cluster's histograms through distributed
//            shared memory and takes the same decision, one cluster barrier a digit;
//   write    a scan over the slice gives each page its place, among those that stay or among the evicted; the list of
//            the pages that stay takes the keys' room, and the weights move along it.
constexpr int kEvThreads = 1024;
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxSlice = 51200;  // 4 bytes a page: 200 KB of shared memory

struct EvictParams {
    const int32_t *table, *seqlens;
    const float *w;
    int64_t bt_stride, w_sb, w_sh, n_pages, W, budget, init, local;
    int32_t shift, Hk;
    int32_t *new_table, *new_lens, *evicted;
    float *new_w;
};

__device__ __forceinline__ uint32_t order_key(float x) {
    if (isnan(x)) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}

__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void cluster_barrier() {
    cluster_arrive();
    cluster_wait();
}

// A 32-bit word of another block's shared memory.
__device__ __forceinline__ uint32_t ld_cluster(const void *mine, uint32_t rank) {
    uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(mine)), v;
    asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(a) : "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// Exclusive scan of one value a thread over the block, and the block's total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    uint32_t s = warp_sums[lane];  // 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    total = __shfl_sync(0xffffffffu, s, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, s, (warp + 31) & 31);
    __syncthreads();  // warp_sums is used again
    return x - v + (warp ? before : 0);
}

__global__ void __launch_bounds__(kEvThreads, 1) evict_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ uint32_t keys[];  // this block's slice; later the list of pages that stay
    __shared__ uint32_t hist[4][256], all[256];
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t found[2];    // the digit, and how many are still wanted inside it
    __shared__ uint32_t slice_kept;
    const uint32_t rank = cluster_rank(), C = cluster_size();
    const int64_t b = blockIdx.x / C;
    const int32_t P = 1 << p.shift;
    int64_t len = __ldg(p.seqlens + b);
    len = len < 0 ? 0 : (len > p.n_pages * P ? p.n_pages * P : len);
    const int64_t used = (len + P - 1) >> p.shift;
    const int64_t drop = used > p.budget ? used - p.budget : 0;
    const int64_t cand0 = p.init, cand1 = used - p.local;  // the pages that may go (only where drop > 0)
    const int64_t per = (used + C - 1) / C;
    const int64_t s0 = per * rank < used ? per * rank : used;
    const int64_t s1 = s0 + per < used ? s0 + per : used;
    const int32_t n = (int32_t)(s1 - s0);
    const float *wb = p.w + b * p.w_sb;
    float *nwb = p.new_w + b * (int64_t)p.Hk * p.W;
    const int32_t *trow = p.table + b * p.bt_stride;
    int32_t *nrow = p.new_table + b * p.n_pages, *erow = p.evicted + b * p.n_pages;
    const int tid = threadIdx.x, lane = tid & 31;
    int64_t kept_before = s0;  // pages that stay, of the slices before this one
    int32_t kept = n;

    if (drop > 0) {
        for (int i = tid; i < 4 * 256; i += kEvThreads) (&hist[0][0])[i] = 0;
        __syncthreads();
        // keys; `per_page` lanes share a page
        const int per_page = P < 32 ? P : 32;
        const int sub = tid & (per_page - 1);
        for (int32_t i0 = 0; i0 < n; i0 += kEvThreads / per_page) {
            const int32_t i = i0 + tid / per_page;
            double sum = 0.0;
            if (i < n) {
                const int64_t at = (s0 + i) << p.shift;
                for (int32_t h = 0; h < p.Hk; ++h)
                    for (int32_t j = sub; j < P; j += per_page)
                        if (at + j < len) sum += (double)__ldg(wb + h * p.w_sh + at + j);
            }
            for (int o = per_page >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (i < n && sub == 0) {
                const uint32_t key = order_key((float)sum);
                keys[i] = key;
                if (s0 + i >= cand0 && s0 + i < cand1) atomicAdd(&hist[0][key >> 24], 1u);
            }
        }
        // the key of the lightest page that stays, digit by digit
        uint32_t prefix = 0;
        uint32_t want = (uint32_t)(cand1 - cand0 - drop);  // candidates that stay
        const bool any = want > 0;
        for (int d = 0; d < 4 && any; ++d) {
            const int sh = 24 - 8 * d;
            if (d > 0) {
                __syncthreads();
                for (int32_t i = tid; i < n; i += kEvThreads) {
                    const uint32_t key = keys[i];
                    if ((key >> (sh + 8)) == prefix && s0 + i >= cand0 && s0 + i < cand1)
                        atomicAdd(&hist[d][(key >> sh) & 255u], 1u);
                }
            }
            cluster_barrier();
            if (tid < 256) {
                uint32_t c = 0;
                for (uint32_t r = 0; r < C; ++r) c += ld_cluster(&hist[d][tid], r);
                all[tid] = c;
            }
            __syncthreads();
            if (tid < 32) {  // lane l has digits 255 - 8l .. 248 - 8l: a scan from the top
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    c[e] = all[255 - 8 * lane - e];
                    sum += c[e];
                }
                uint32_t above = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, above, o);
                    if (lane >= o) above += y;
                }
                above -= sum;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (above < want && want <= above + c[e]) {
                        found[0] = 255 - 8 * lane - e;
                        found[1] = want - above;
                    }
                    above += c[e];
                }
            }
            __syncthreads();
            prefix = (prefix << 8) | found[0];
            want = found[1];
        }
        // pages of exactly that key: `want` of them stay, the first ones
        uint32_t eq_left = 0, eq_here = 0;
        if (any) {
            uint32_t eq_before = 0;
            for (uint32_t r = 0; r < rank; ++r) eq_before += ld_cluster(&hist[3][prefix & 255u], r);
            eq_here = hist[3][prefix & 255u];
            eq_left = want > eq_before ? want - eq_before : 0;
            eq_left = eq_left < eq_here ? eq_left : eq_here;
        }
        auto sure = [&](int32_t i) {
            const int64_t e = s0 + i;
            return e < cand0 || e >= cand1 || (any && keys[i] > prefix);
        };
        uint32_t n_sure = 0;
        for (int32_t i = tid; i < n; i += kEvThreads) n_sure += sure(i);
        uint32_t total;
        block_scan(n_sure, warp_sums, total);
        if (tid == 0) slice_kept = total + eq_left;
        kept = (int32_t)(total + eq_left);
        cluster_barrier();
        kept_before = 0;
        for (uint32_t r = 0; r < rank; ++r) kept_before += ld_cluster(&slice_kept, r);
        cluster_arrive();  // waited for at the end: no block leaves while another reads its shared memory
        // places: among those that stay, or among the evicted
        uint32_t base = 0, eq_base = 0;
        for (int32_t i0 = 0; i0 < n; i0 += kEvThreads) {
            const int32_t i = i0 + tid;
            const bool is_sure = i < n && sure(i);
            const bool eq = i < n && !is_sure && any && keys[i] == prefix;
            uint32_t n_eq, n_stay;
            const uint32_t eq_at = block_scan(eq ? 1u : 0u, warp_sums, n_eq) + eq_base;
            const bool stay = is_sure || (eq && eq_at < eq_left);
            const uint32_t at = block_scan(stay ? 1u : 0u, warp_sums, n_stay) + base;
            if (i < n) {
                const int32_t page = __ldg(trow + s0 + i);
                if (stay) {
                    keys[at] = (uint32_t)i;  // at <= i: this chunk's keys have been read
                    nrow[kept_before + at] = page;
                } else {
                    erow[s0 - kept_before + i - at] = page;
                }
            }
            base += n_stay;
            eq_base += n_eq;
        }
        __syncthreads();
    } else {
        for (int32_t i = tid; i < n; i += kEvThreads) {
            keys[i] = (uint32_t)i;
            nrow[s0 + i] = __ldg(trow + s0 + i);
        }
        __syncthreads();
    }
    // the weights of the pages that stay
    const int64_t m = (int64_t)kept << p.shift;
    for (int64_t j = tid; j < m; j += kEvThreads) {
        const int64_t at = ((s0 + keys[j >> p.shift]) << p.shift) + (j & (P - 1));
        float *dst = nwb + (kept_before << p.shift) + j;
        for (int32_t h = 0; h < p.Hk; ++h) dst[h * p.W] = at < len ? __ldg(wb + h * p.w_sh + at) : 0.0f;
    }
    // behind them: pages of the row that are not in use yet move up, and nothing fills the rest
    const int64_t me = (int64_t)rank * kEvThreads + tid, all_threads = (int64_t)C * kEvThreads;
    for (int64_t e = used + me; e < p.n_pages; e += all_threads) nrow[e - drop] = __ldg(trow + e);
    for (int64_t e = me; e < drop; e += all_threads) nrow[p.n_pages - drop + e] = -1;
    for (int64_t e = drop + me; e < p.n_pages; e += all_threads) erow[e] = -1;
    for (int64_t j = ((used - drop) << p.shift) + me; j < p.W; j += all_threads)
        for (int32_t h = 0; h < p.Hk; ++h) nwb[h * p.W + j] = 0.0f;
    if (rank == 0 && tid == 0) p.new_lens[b] = (int32_t)(len - (drop << p.shift));
    if (drop > 0) cluster_wait();
}

bool power_of_two(int64_t x) { return x > 0 && (x & (x - 1)) == 0; }

int log2_of(int64_t x) {
    int s = 0;
    while (((int64_t)1 << s) < x) ++s;
    return s;
}

}  // namespace

extern "C" int unum_cache_append(const void *k, const void *v, int64_t T, int64_t Hk, int64_t D, int64_t k_st,
                                 int64_t k_sh, int64_t v_st, int64_t v_sh, void *k_cache, void *v_cache,
                                 int64_t n_tokens, int64_t kc_st, int64_t kc_sh, int64_t vc_st, int64_t vc_sh,
                                 const int32_t *block_table, int64_t B, int64_t n_pages, int64_t bt_stride,
                                 int64_t page_size, const int32_t *token_to_bs, const int32_t *token_pos_in_bs,
                                 void *stream) {
    unum::clear_error();
    UNUM_CHECK_ARG(T >= 0 && Hk > 0 && B >= 0 && n_pages >= 0 && n_tokens >= 0, "bad sizes");
    if (D != 64 && D != 128) {
        unum::set_error("head_dim %lld not supported (64 or 128)", (long long)D);
        return UNUM_ERR_UNSUPPORTED;
    }
    UNUM_CHECK_ARG(power_of_two(page_size) && page_size <= 65536, "page_size must be a power of two up to 65536 (got %lld)",
                   (long long)page_size);
    if (T == 0 || B == 0 || n_pages == 0 || n_tokens == 0) return UNUM_OK;
    UNUM_CHECK_ARG(k && v && k_cache && v_cache && block_table && token_to_bs && token_pos_in_bs,
                   "null pointer argument");
    UNUM_CHECK_ARG(unum::aligned16(k) && unum::aligned16(v) && unum::aligned16(k_cache) && unum::aligned16(v_cache),
                   "k, v, k_cache and v_cache must be 16-byte aligned");
    UNUM_CHECK_ARG((k_st | k_sh | v_st | v_sh | kc_st | kc_sh | vc_st | vc_sh) % 8 == 0,
                   "strides of k, v, k_cache and v_cache must be multiples of 8 elements");
    AppendParams p;
    p.k = (const uint8_t *)k;
    p.v = (const uint8_t *)v;
    p.kc = (uint8_t *)k_cache;
    p.vc = (uint8_t *)v_cache;
    p.k_st = 2 * k_st, p.k_sh = 2 * k_sh, p.v_st = 2 * v_st, p.v_sh = 2 * v_sh;
    p.kc_st = 2 * kc_st, p.kc_sh = 2 * kc_sh, p.vc_st = 2 * vc_st, p.vc_sh = 2 * vc_sh;
    p.table = block_table;
    p.bs = token_to_bs;
    p.pos = token_pos_in_bs;
    p.bt_stride = bt_stride;
    p.n_pages = n_pages;
    p.n_tokens = n_tokens;
    p.T = T;
    p.B = B;
    p.shift = log2_of(page_size);
    p.hchunks_shift = log2_of(D / 8);
    UNUM_CHECK_ARG(Hk <= 65536, "too many kv heads");
    p.chunks = (int32_t)(Hk * (D / 8));
    const int64_t blocks = (T * p.chunks + 255) / 256;
    UNUM_CHECK_ARG(T < ((int64_t)1 << 40) && blocks < ((int64_t)1 << 31), "too many tokens");
    append_kernel<<<(unsigned)blocks, 256, 0, (cudaStream_t)stream>>>(p);
    return unum::check_launch("append_kernel");
}

extern "C" int unum_cache_evict(const int32_t *block_table, int64_t B, int64_t n_pages, int64_t bt_stride,
                                const int32_t *seqlens, const float *weights, int64_t Hk, int64_t w_sb, int64_t w_sh,
                                int64_t page_size, int64_t budget, int64_t init_pages, int64_t local_pages,
                                int32_t *new_table, int32_t *new_seqlens, float *new_weights, int32_t *evicted,
                                void *stream) {
    unum::clear_error();
    UNUM_CHECK_ARG(B >= 0 && n_pages >= 0 && Hk > 0 && Hk <= 65536, "bad sizes");
    UNUM_CHECK_ARG(power_of_two(page_size) && page_size <= 65536, "page_size must be a power of two up to 65536 (got %lld)",
                   (long long)page_size);
    UNUM_CHECK_ARG(init_pages >= 0 && local_pages >= 1, "init_pages must be >= 0 and local_pages >= 1 (got %lld, %lld)",
                   (long long)init_pages, (long long)local_pages);
    UNUM_CHECK_ARG(budget >= init_pages && budget - init_pages >= local_pages,
                   "budget must hold init_pages + local_pages (got %lld < %lld + %lld)", (long long)budget,
                   (long long)init_pages, (long long)local_pages);
    if (B == 0) return UNUM_OK;
    if (n_pages > kMaxCluster * kMaxSlice) {
        unum::set_error("at most %lld pages a sequence (got %lld)", (long long)(kMaxCluster * kMaxSlice),
                        (long long)n_pages);
        return UNUM_ERR_UNSUPPORTED;
    }
    UNUM_CHECK_ARG(n_pages * page_size < ((int64_t)1 << 31), "n_pages * page_size must stay below 2^31");
    UNUM_CHECK_ARG(B < ((int64_t)1 << 28), "too many sequences");
    UNUM_CHECK_ARG(seqlens && new_seqlens, "null pointer argument");
    UNUM_CHECK_ARG(n_pages == 0 || (block_table && weights && new_table && new_weights && evicted),
                   "null pointer argument");
    EvictParams p;
    p.table = block_table;
    p.seqlens = seqlens;
    p.w = weights;
    p.bt_stride = bt_stride;
    p.w_sb = w_sb;
    p.w_sh = w_sh;
    p.n_pages = n_pages;
    p.W = n_pages * page_size;
    p.budget = budget;
    p.init = init_pages;
    p.local = local_pages;
    p.shift = log2_of(page_size);
    p.Hk = (int32_t)Hk;
    p.new_table = new_table;
    p.new_lens = new_seqlens;
    p.evicted = evicted;
    p.new_w = new_weights;
    int C = 1;
    while (C < kMaxCluster && n_pages > C * kMaxSlice) C *= 2;
    const int64_t slice = (n_pages + C - 1) / C;
    const size_t smem = (size_t)(slice < 1 ? 1 : slice) * 4;
    UNUM_CHECK_CUDA(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(kMaxSlice * 4)));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)C;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, evict_kernel, p));
    return unum::check_launch("evict_kernel");
}
