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
//   gathered, taken in 64 bits and rounded to 32 once: another order of summation gives another weight only where the
//   sum lies within a few 2^-53 of its terms from a border of the rounding.  Ties go to the lower index and a NaN ranks
//   below every number.  The row closes up over what is evicted.
#include <cuda_runtime.h>

#include "common.cuh"
#include "sm100.cuh"

namespace {

using namespace unum::sm100;

// ------------------------------------------------------------------------------------------------ append
// One thread moves the same 16 bytes of the key and of the value row.  The rows' loads do not wait for the
// table's, and 2048 threads an SM keep 64 KB in flight, which covers HBM's latency.  131072 tokens of 2 x 128 (268 MB)
// take 42.9 us, 6.26 TB/s, as long as a plain copy; 53.8 us without the streaming hint on the stores, 44.4 us with two
// pieces a thread.
struct AppendParams {
    const uint8_t *k, *v;
    uint8_t *kc, *vc;
    int64_t k_st, k_sh, v_st, v_sh, kc_st, kc_sh, vc_st, vc_sh;  // bytes
    const int32_t *table, *bs, *pos;
    int64_t bt_stride, n_pages, n_tokens, T, B;
    int32_t shift, chunks, hchunks_shift;  // 16-byte pieces of a token's row over all heads; log2 of one head's
};

__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
    unum::wait_for_previous_kernel();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t t = i / p.chunks;
    if (t >= p.T) return;
    const int32_t c = (int32_t)(i - t * p.chunks);
    const int64_t h = c >> p.hchunks_shift, o = (int64_t)(c & ((1 << p.hchunks_shift) - 1)) * 16;
    const int4 kv = __ldcs(reinterpret_cast<const int4 *>(p.k + t * p.k_st + h * p.k_sh + o));
    const int4 vv = __ldcs(reinterpret_cast<const int4 *>(p.v + t * p.v_st + h * p.v_sh + o));
    const int64_t b = p.bs[t], at = (int64_t)p.pos[t] - 1;
    if (b < 0 || b >= p.B || at < 0 || (at >> p.shift) >= p.n_pages) return;
    if (at == INT32_MAX - 1) return;  // the largest count stands for all that 32 bits do not hold
    const int64_t page = p.table[b * p.bt_stride + (at >> p.shift)];
    const int64_t token = (page << p.shift) + (at & ((1 << p.shift) - 1));
    if (page < 0 || token >= p.n_tokens) return;
    __stcs(reinterpret_cast<int4 *>(p.kc + token * p.kc_st + h * p.kc_sh + o), kv);
    __stcs(reinterpret_cast<int4 *>(p.vc + token * p.vc_st + h * p.vc_sh + o), vv);
}

// ------------------------------------------------------------------------------------------------ evict
// One cluster of C blocks for each sequence; block r has a contiguous slice of its pages in use, with one 32-bit key
// a page in shared memory (the float's bits in an order that compares as unsigned; 0 = NaN).
//   keys     the sums, four pages a thread (or group of threads) under way at once;
//   select   radix selection over four 8-bit digits.  Keys crowd into few bins of the first, so a block counts in eight
//            histograms by lane.  After a cluster barrier every block adds up the cluster's counts through distributed
//            shared memory and takes the same decision; where all pages of the digit found are wanted, it is the last
//            one (mostly the third for long sequences, the second or third for short ones).  (Adding them up with remote atomics took 13 us a digit with 16
//            blocks: they are served one at a time.)
//   write    each warp has a contiguous part of the slice; a count and one scan over the warps give each page its
//            place, among those that stay or among the evicted, and the weights move along.
// Where the first and the last pages fill the budget nothing is chosen: no sums are taken, and places go by the index alone.
// What is filled behind the new ends does not wait for any of it and is written first.
// Bound by latency for one sequence (the barriers), by HBM for a batch.
constexpr int kEvThreads = 512;  // with 1024, block barriers cost more than the added warps hid (12.5 against 10.3 us)
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int64_t kMaxSlice = 25600;  // 4 bytes a page: 100 KB of shared memory
constexpr int64_t kMaxPages = kMaxCluster * kMaxSlice;
constexpr int kBins = 256;
constexpr int kGroups = 2 * kEvThreads / kBins;
constexpr int kCopies = 8;   // of the histogram
constexpr int kBatch = 4;    // loads of a thread under way

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

// Exclusive scan over the block's warps of a value that each warp's lanes agree on, and the total.
__device__ __forceinline__ uint32_t scan_warps(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();  // warp_sums may still be read
    if (lane == 0) warp_sums[warp] = v;
    __syncthreads();
    const uint32_t x = lane < kEvWarps ? warp_sums[lane] : 0;
    total = __reduce_add_sync(0xffffffffu, x);
    return __reduce_add_sync(0xffffffffu, lane < warp ? x : 0);
}

// kVec: pages of 4 positions and more whose weights 16-byte loads can read.
template <bool kVec> __global__ void __launch_bounds__(kEvThreads, 2) evict_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ uint32_t keys[];  // this block's slice
    __shared__ __align__(8) uint32_t hist[kCopies][kBins];
    __shared__ uint32_t counts[4][kBins / 2];             // this block's, of each digit
    __shared__ __align__(8) uint32_t sums[kGroups][kBins];  // the cluster's, of every kGroups-th block
    __shared__ uint32_t warp_sums[kEvWarps];
    __shared__ uint32_t found[3];    // the digit, how many are still wanted with it, and how many have it
    __shared__ uint32_t slice_eq, slice_sure;
    unum::wait_for_previous_kernel();
    const uint32_t rank = cluster_ctarank(), C = cluster_nctarank();
    const int64_t b = blockIdx.x / C;
    const int32_t P = 1 << p.shift;
    int64_t len = p.seqlens[b];
    len = len < 0 ? 0 : (len > p.n_pages * P ? p.n_pages * P : len);
    const int64_t used = (len + P - 1) >> p.shift;
    const int64_t drop = used > p.budget ? used - p.budget : 0;
    const int64_t per = (used + C - 1) / C;
    const int64_t s0 = per * rank < used ? per * rank : used;
    const int64_t s1 = s0 + per < used ? s0 + per : used;
    const int32_t n = (int32_t)(s1 - s0);
    // the pages that may go (only where drop > 0), within the slice
    const int64_t c0 = p.init - s0, c1 = used - p.local - s0;
    const int32_t cand0 = (int32_t)(c0 < 0 ? 0 : (c0 > n ? n : c0)), cand1 = (int32_t)(c1 < 0 ? 0 : (c1 > n ? n : c1));
    const float *wb = p.w + b * p.w_sb;
    float *nwb = p.new_w + b * (int64_t)p.Hk * p.W;
    const int32_t *trow = p.table + b * p.bt_stride;
    int32_t *nrow = p.new_table + b * p.n_pages, *erow = p.evicted + b * p.n_pages;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // a warp's part of the slice
    const int32_t part = ((n + kEvWarps - 1) / kEvWarps + 31) / 32 * 32;
    const int32_t i0 = min(warp * part, n), i1 = min(i0 + part, n);
    // pages that stay: of the slices before this one, and of this slice before the warp's part
    int64_t kept_before = s0;
    uint32_t stay_at = i0;
    // keys from edge_from on stay; of those equal to edge, eq_left (eq_at: so far)
    uint32_t edge = 0, edge_from = 0, eq_at = 0, eq_left = 0;

    // behind what stays: pages of the row that are not in use yet move up, and nothing fills the rest
    const int64_t me = (int64_t)rank * kEvThreads + tid, all_threads = (int64_t)C * kEvThreads;
    for (int64_t e = used + me; e < p.n_pages; e += all_threads) nrow[e - drop] = trow[e];
    for (int64_t e = me; e < drop; e += all_threads) nrow[p.n_pages - drop + e] = -1;
    for (int64_t e = drop + me; e < p.n_pages; e += all_threads) erow[e] = -1;
    const int64_t end = (used - drop) << p.shift;
    if (p.W % 4 == 0) {
        const int64_t end4 = (end + 3) / 4 * 4;
        for (int32_t h = 0; h < p.Hk; ++h) {
            float *row = nwb + h * p.W;
            for (int64_t j = end4 + 4 * me; j < p.W; j += 4 * all_threads)
                __stcs(reinterpret_cast<float4 *>(row + j), make_float4(0.0f, 0.0f, 0.0f, 0.0f));
            if (me < end4 - end) row[end + me] = 0.0f;
        }
    } else {
        for (int32_t h = 0; h < p.Hk; ++h)
            for (int64_t j = end + me; j < p.W; j += all_threads) nwb[h * p.W + j] = 0.0f;
    }

    if (drop > 0) {
        uint32_t want = (uint32_t)(p.budget - p.init - p.local);  // pages that stay by their weight
        uint32_t prefix = 0xffffffffu, all_from = 0xffffffffu;    // no key is that large
        if (want > 0) {
            for (int i = tid; i < kCopies * kBins; i += kEvThreads) (&hist[0][0])[i] = 0;
            __syncthreads();
            // keys; `lanes` threads share a page
            constexpr int kWide = kVec ? 4 : 1;
            const int lanes = P < 32 * kWide ? P / kWide : 32;
            const int sub = (tid & (lanes - 1)) * kWide;
            const int32_t stride = kEvThreads / lanes;
            uint32_t *my_hist = hist[lane & (kCopies - 1)];
            if (lanes >= kCopies) my_hist = hist[(tid / lanes) & (kCopies - 1)];
            for (int32_t i00 = tid / lanes; i00 < n + tid / lanes; i00 += kBatch * stride) {
                double sum[kBatch] = {};
                for (int32_t j = sub; j < P; j += lanes * kWide) {
    #pragma unroll 2
                    for (int32_t h = 0; h < p.Hk; ++h) {
                        const float *src = wb + h * p.w_sh + (s0 << p.shift) + j;
                        if (kVec) {
                            float4 v[kBatch];
    #pragma unroll
                            for (int e = 0; e < kBatch; ++e)
                                if (i00 + e * stride < n)
                                    v[e] = *reinterpret_cast<const float4 *>(src + ((int64_t)(i00 + e * stride) << p.shift));
    #pragma unroll
                            for (int e = 0; e < kBatch; ++e) {
                                const int64_t left = len - ((s0 + i00 + e * stride) << p.shift) - j;
                                if (left >= 4) {
                                    sum[e] += ((double)v[e].x + (double)v[e].y) + ((double)v[e].z + (double)v[e].w);
                                } else {
                                    if (left > 0) sum[e] += (double)v[e].x;
                                    if (left > 1) sum[e] += (double)v[e].y;
                                    if (left > 2) sum[e] += (double)v[e].z;
                                }
                            }
                        } else {
                            float v[kBatch];
    #pragma unroll
                            for (int e = 0; e < kBatch; ++e) {
                                const int64_t at = ((int64_t)(i00 + e * stride) << p.shift);
                                v[e] = i00 + e * stride < n && (s0 << p.shift) + at + j < len ? src[at] : 0.0f;
                            }
    #pragma unroll
                            for (int e = 0; e < kBatch; ++e) sum[e] += (double)v[e];
                        }
                    }
                }
    #pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    for (int o = lanes >> 1; o > 0; o >>= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
                    const int32_t i = i00 + e * stride;
                    if (i < n && sub == 0) {
                        const uint32_t key = order_key((float)sum[e]);
                        keys[i] = key;
                        if (i >= cand0 && i < cand1) atomicAdd(&my_hist[key >> 24], 1u);
                    }
                }
            }
            // the key of the lightest page that stays, digit by digit
            prefix = 0;
            my_hist = hist[lane & (kCopies - 1)];
            for (int d = 0; d < 4; ++d) {
                const int sh = 24 - 8 * d;
                if (d > 0) {
    #pragma unroll 4
                    for (int32_t i = cand0 + tid; i < cand1; i += kEvThreads) {
                        const uint32_t key = keys[i];
                        if ((key >> (sh + 8)) == prefix) atomicAdd(&my_hist[(key >> sh) & 255u], 1u);
                    }
                }
                __syncthreads();
                if (tid < kBins / 2) {  // two counts a word: a slice has fewer pages than 2^16
                    uint32_t c = 0;
    #pragma unroll
                    for (int i = 0; i < kCopies; ++i) {
                        const uint2 h = *reinterpret_cast<uint2 *>(&hist[i][2 * tid]);
                        c += h.x | h.y << 16;
                        *reinterpret_cast<uint2 *>(&hist[i][2 * tid]) = make_uint2(0, 0);
                    }
                    counts[d][tid] = c;
                }
                if (C > 1) cluster_sync();
                else __syncthreads();
                {
                    const int pair = tid % (kBins / 2), group = tid / (kBins / 2);
                    uint32_t c0 = 0, c1 = 0;
    #pragma unroll 4
                    for (uint32_t r = group; r < C; r += kGroups) {
                        const uint32_t c = C > 1 ? ld_cluster_u32(peer_smem(&counts[d][pair], r)) : counts[d][pair];
                        c0 += c & 0xffffu;
                        c1 += c >> 16;
                    }
                    *reinterpret_cast<uint2 *>(&sums[group][2 * pair]) = make_uint2(c0, c1);
                }
                __syncthreads();
                if (warp == 0) {  // lane l has digits 255 - 8l .. 248 - 8l: a scan from the top
                    uint32_t c[8], sum = 0;
    #pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        c[e] = 0;
    #pragma unroll
                        for (int i = 0; i < kGroups; ++i) c[e] += sums[i][255 - 8 * lane - e];
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
                            found[2] = c[e];
                        }
                        above += c[e];
                    }
                }
                __syncthreads();
                prefix = (prefix << 8) | found[0];
                want = found[1];
                all_from = prefix << sh;
                if (found[2] == want) {  // all of them
                    prefix = 0xffffffffu;
                    break;
                }
                if (d == 3) ++all_from;
            }
        } else {
            for (int32_t i = i0 + lane; i < i1; i += 32) keys[i] = 0;  // read below by the lane that writes it
        }
        // Keys from all_from on stay, and of the pages with the key `prefix` the first `want`.  What this warp's part has
        // of either:
        uint32_t n_sure = 0, n_eq = 0;
        for (int32_t i = i0 + lane; i < i1; i += 32) {
            const uint32_t key = keys[i];
            const bool s = i < cand0 || i >= cand1 || key >= all_from;
            n_sure += s;
            n_eq += !s && key == prefix;
        }
        n_sure = __reduce_add_sync(0xffffffffu, n_sure);
        n_eq = __reduce_add_sync(0xffffffffu, n_eq);
        uint32_t all_sure, all_eq;
        const uint32_t sure_at = scan_warps(n_sure, warp_sums, all_sure);
        eq_at = scan_warps(n_eq, warp_sums, all_eq);
        if (tid == 0) {
            slice_eq = all_eq;
            slice_sure = all_sure;
        }
        if (C > 1) cluster_sync();
        // slices before this one: their pages of that key come first
        uint32_t eq_before = 0, sure_before = 0;
        for (uint32_t r = 0; r < rank; ++r) {
            eq_before += ld_cluster_u32(peer_smem(&slice_eq, r));
            sure_before += ld_cluster_u32(peer_smem(&slice_sure, r));
        }
        if (C > 1) cluster_arrive();  // waited for at the end: no block leaves while another reads its shared memory
        eq_left = want - min(eq_before, want);  // of this slice's, the first ones
        kept_before = sure_before + min(eq_before, want);
        stay_at = sure_at + min(eq_at, eq_left);
        edge = prefix;
        edge_from = all_from;
    }
    // places.  The warp's list of pages that stay takes the room of its keys, behind where it reads.
    const int64_t to = (kept_before + stay_at) << p.shift;
    int32_t m = 0, page = i0 + lane < i1 ? trow[s0 + i0 + lane] : 0;
#pragma unroll 1
    for (int32_t j0 = i0; j0 < i1; j0 += 32) {
        const int32_t i = j0 + lane, my_page = page;
        if (i + 32 < i1) page = trow[s0 + i + 32];
        const uint32_t below = (1u << lane) - 1;
        bool stay = i < i1;
        if (drop > 0) {
            const uint32_t key = stay ? keys[i] : 0;
            const bool sure = stay && (i < cand0 || i >= cand1 || key >= edge_from);
            const bool eq = stay && !sure && key == edge;
            const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
            stay = sure || (eq && eq_at + __popc(eqs & below) < eq_left);
            eq_at += __popc(eqs);
        }
        const uint32_t stays = __ballot_sync(0xffffffffu, stay);
        const int32_t at = m + __popc(stays & below);
        if (stay) {
            nrow[kept_before + stay_at + at] = my_page;
            keys[i0 + at] = (uint32_t)i;
        } else if (i < i1) {
            erow[s0 + i - kept_before - stay_at - at] = my_page;
        }
        m += __popc(stays);
    }
    __syncwarp();
    // and the weights of those pages
    m <<= p.shift;
    {
        constexpr int kWide = kVec ? 4 : 1;
        for (int32_t q0 = lane * kWide; q0 < m; q0 += 32 * kWide * kBatch) {
            int64_t from[kBatch];
#pragma unroll
            for (int e = 0; e < kBatch; ++e) {
                const int32_t q = q0 + 32 * kWide * e;
                from[e] = q < m ? ((s0 + keys[i0 + (q >> p.shift)]) << p.shift) + (q & (P - 1)) : len;
            }
#pragma unroll 2
            for (int32_t h = 0; h < p.Hk; ++h) {
                const float *src = wb + h * p.w_sh;
                float *dst = nwb + h * p.W + to + q0;
                if (kVec) {
                    float4 v[kBatch];
#pragma unroll
                    for (int e = 0; e < kBatch; ++e)
                        v[e] = from[e] < len ? *reinterpret_cast<const float4 *>(src + from[e])
                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        // behind the length: zero, whatever is there
                        if (from[e] + 1 >= len) v[e].y = 0.0f;
                        if (from[e] + 2 >= len) v[e].z = 0.0f;
                        if (from[e] + 3 >= len) v[e].w = 0.0f;
                        if (q0 + 128 * e < m) __stcs(reinterpret_cast<float4 *>(dst + 128 * e), v[e]);
                    }
                } else {
                    float v[kBatch];
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) v[e] = from[e] < len ? src[from[e]] : 0.0f;
#pragma unroll
                    for (int e = 0; e < kBatch; ++e)
                        if (q0 + 32 * e < m) __stcs(dst + 32 * e, v[e]);
                }
            }
        }
    }
    if (rank == 0 && tid == 0) p.new_lens[b] = (int32_t)(len - (drop << p.shift));
    if (drop > 0 && C > 1) cluster_wait();
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
    cudaLaunchAttribute attr = unum::behind_previous_kernel();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, append_kernel, p));
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
    if (n_pages > kMaxPages) {
        unum::set_error("at most %lld pages a sequence (got %lld)", (long long)kMaxPages, (long long)n_pages);
        return UNUM_ERR_UNSUPPORTED;
    }
    UNUM_CHECK_ARG(n_pages * page_size < ((int64_t)1 << 30), "n_pages * page_size must stay below 2^30");
    UNUM_CHECK_ARG(B < ((int64_t)1 << 28), "too many sequences");
    UNUM_CHECK_ARG(seqlens && new_seqlens, "null pointer argument");
    UNUM_CHECK_ARG(n_pages == 0 || (block_table && weights && new_table && new_weights && evicted),
                   "null pointer argument");
    UNUM_CHECK_ARG(unum::aligned16(new_weights), "new_weights must be 16-byte aligned");
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
    // As many blocks a sequence as keep the whole batch resident (two an SM), while each still has 4096 weights or more.
    int64_t C = 1;
    while (C < kMaxCluster && (n_pages > C * kMaxSlice || (B * C * 2 <= 2 * unum::sm_count() &&
                                                           n_pages * page_size * Hk >= C * 2 * 4096)))
        C *= 2;
    const int64_t slice = (n_pages + C - 1) / C;
    const size_t smem = (size_t)(slice < 1 ? 1 : slice) * 4;
    const bool vec = page_size >= 4 && (w_sb | w_sh) % 4 == 0 && unum::aligned16(weights);
    auto *kernel = vec ? evict_kernel<true> : evict_kernel<false>;
    UNUM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMaxSlice * 4)));
    UNUM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * C));
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1] = unum::behind_previous_kernel();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return unum::check_launch("evict_kernel");
}
