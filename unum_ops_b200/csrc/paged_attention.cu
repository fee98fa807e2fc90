// Attention of one new token for each sequence over its paged key-value cache.
//
// The reference has no dense attention over the cache; its get_block_table
// (src/unum_ops/sparse_kernel_extension/get_table_torch.py:29-44) fixes how a table maps positions to tokens.  For
// sequence b, query head h of kv head g = h / G and position p (page size P, a power of two):
//     token(p) = table[b, p / P] * P + p % P,   valid iff p < len_b and 0 <= token < n_tokens
//     s_p = scale * q[b,h] . k[token(p), g];   lse = log sum_p exp(s_p);   out = sum_p exp(s_p - lse) v[token(p), g]
//     weights[b,g,p] += sum over the group's heads of exp(s_p - lse)          (where they are gathered)
// A row without a valid position is 0 with lse = -inf.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

constexpr int kTile = 32;
constexpr int kThreads = 256;
constexpr int kMaxG = 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
    const void *q, *kc, *vc;
    int64_t q_sb, q_sh, k_st, k_sh, v_st, v_sh;
    const int32_t *table, *lens;
    int64_t bt_stride, n_tokens, max_len;
    int32_t shift, Hk, G;
    float c;  // scale * log2(e)
    void *out;
    float *lse, *weights;
    int64_t w_sb, w_sh;
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }

// The simplest right form: one block for each (sequence, kv head), products on the CUDA cores.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attend_kernel(const __grid_constant__ Params p) {
    extern __shared__ float sm[];
    const int G = p.G;
    float *q = sm, *o = q + G * D, *kv = o + G * D, *s = kv + kTile * (D + 1), *m = s + G * kTile, *l = m + G, *f = l + G;
    __shared__ int64_t tok[kTile];
    const int g = blockIdx.x, tid = threadIdx.x;
    const int64_t b = blockIdx.y;
    const T *qp = (const T *)p.q, *kc = (const T *)p.kc + g * p.k_sh, *vc = (const T *)p.vc + g * p.v_sh;
    int64_t len = p.lens[b];
    len = len < 0 ? 0 : (len > p.max_len ? p.max_len : len);
    for (int i = tid; i < G * D; i += kThreads) {
        q[i] = to_f(qp[b * p.q_sb + (int64_t)(g * G + i / D) * p.q_sh + i % D]);
        o[i] = 0.f;
    }
    for (int i = tid; i < G; i += kThreads) m[i] = -INFINITY, l[i] = 0.f;
    auto load = [&](const T *c, int64_t st) {
        for (int i = tid; i < kTile * D; i += kThreads) {
            const int64_t t = tok[i / D];
            kv[i / D * (D + 1) + i % D] = t >= 0 ? to_f(c[t * st + i % D]) : 0.f;
        }
    };
    auto scores = [&](int64_t p0) {
        __syncthreads();
        if (tid < kTile) {
            const int64_t at = p0 + tid;
            int64_t t = -1;
            if (at < len) {
                const int64_t page = p.table[b * p.bt_stride + (at >> p.shift)];
                t = (page << p.shift) + (at & ((1 << p.shift) - 1));
                if (page < 0 || t >= p.n_tokens) t = -1;
            }
            tok[tid] = t;
        }
        __syncthreads();
        load(kc, p.k_st);
        __syncthreads();
        for (int i = tid; i < G * kTile; i += kThreads) {
            const int h = i / kTile, j = i % kTile;
            float x = 0.f;
            for (int d = 0; d < D; ++d) x = fmaf(q[h * D + d], kv[j * (D + 1) + d], x);
            s[i] = tok[j] >= 0 ? x * p.c : -INFINITY;
        }
        __syncthreads();
    };
    for (int64_t p0 = 0; p0 < len; p0 += kTile) {
        scores(p0);
        for (int h = tid; h < G; h += kThreads) {
            float mx = m[h];
            for (int j = 0; j < kTile; ++j) mx = fmaxf(mx, s[h * kTile + j]);
            const float base = mx == -INFINITY ? 0.f : mx;
            float sum = 0.f;
            for (int j = 0; j < kTile; ++j) {
                const float e = exp2f(s[h * kTile + j] - base);
                s[h * kTile + j] = e;
                sum += e;
            }
            f[h] = exp2f(m[h] - base);
            l[h] = l[h] * f[h] + sum;
            m[h] = mx;
        }
        load(vc, p.v_st);
        __syncthreads();
        for (int i = tid; i < G * D; i += kThreads) {
            float x = o[i] * f[i / D];
            for (int j = 0; j < kTile; ++j) x = fmaf(s[i / D * kTile + j], kv[j * (D + 1) + i % D], x);
            o[i] = x;
        }
    }
    __syncthreads();
    T *out = (T *)p.out + (b * p.Hk + g) * G * D;
    for (int i = tid; i < G * D; i += kThreads) out[i] = from_f<T>(l[i / D] != 0.f ? o[i] / l[i / D] : 0.f);
    for (int i = tid; i < G; i += kThreads) {
        m[i] = l[i] != 0.f ? m[i] + log2f(l[i]) : -INFINITY;
        if (p.lse) p.lse[(b * p.Hk + g) * G + i] = m[i] * kLn2;
    }
    if (!p.weights) return;
    for (int64_t p0 = 0; p0 < len; p0 += kTile) {
        scores(p0);
        if (tid < kTile && tok[tid] >= 0) {
            float x = 0.f;
            for (int h = 0; h < G; ++h)
                if (m[h] != -INFINITY) x += exp2f(s[h * kTile + tid] - m[h]);
            p.weights[b * p.w_sb + g * p.w_sh + p0 + tid] += x;
        }
    }
}

template <typename T, int D> int launch(const Params &p, int64_t B, cudaStream_t s) {
    const int smem = (2 * p.G * D + kTile * (D + 1) + p.G * kTile + 3 * p.G) * 4;
    UNUM_CHECK_CUDA(cudaFuncSetAttribute(attend_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    attend_kernel<T, D><<<dim3(p.Hk, (unsigned)B), kThreads, smem, s>>>(p);
    return unum::check_launch("attend_kernel");
}

}  // namespace

extern "C" size_t unum_paged_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t max_seqlen,
                                                      int gather_weights) {
    (void)B, (void)Hq, (void)Hk, (void)D, (void)max_seqlen, (void)gather_weights;
    return 16;
}

extern "C" int unum_paged_attention(const void *q, int64_t B, int64_t Hq, int64_t D, int64_t q_sb, int64_t q_sh,
                                    const void *k_cache, const void *v_cache, int dtype, int64_t n_tokens, int64_t Hk,
                                    int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, const int32_t *block_table,
                                    int64_t n_pages, int64_t bt_stride, int64_t page_size, const int32_t *seqlens,
                                    int64_t max_seqlen, float softmax_scale, void *out, float *lse, float *weights,
                                    int64_t w_sb, int64_t w_sh, void *workspace, size_t workspace_bytes,
                                    void *stream) {
    unum::clear_error();
    UNUM_CHECK_ARG(B >= 0 && Hq > 0 && Hk > 0 && n_tokens >= 0 && n_pages >= 0 && max_seqlen >= 0, "bad sizes");
    UNUM_CHECK_ARG(dtype == UNUM_DTYPE_BF16 || dtype == UNUM_DTYPE_F16, "unsupported dtype code %d (bf16 or f16)", dtype);
    UNUM_CHECK_ARG(Hq % Hk == 0, "%lld query heads are no multiple of %lld kv heads", (long long)Hq, (long long)Hk);
    if ((D != 64 && D != 128) || Hq / Hk > kMaxG) {
        unum::set_error("paged attention supports head_dim 64 or 128 and at most %d query heads per kv head "
                        "(got head_dim %lld, %lld/%lld heads)", kMaxG, (long long)D, (long long)Hq, (long long)Hk);
        return UNUM_ERR_UNSUPPORTED;
    }
    UNUM_CHECK_ARG(page_size > 0 && (page_size & (page_size - 1)) == 0 && page_size <= 65536,
                   "page_size must be a power of two up to 65536 (got %lld)", (long long)page_size);
    if (B == 0) return UNUM_OK;
    UNUM_CHECK_ARG(q && seqlens && out, "null pointer argument");
    UNUM_CHECK_ARG(max_seqlen <= n_pages * page_size, "max_seqlen %lld exceeds the table's %lld positions",
                   (long long)max_seqlen, (long long)(n_pages * page_size));
    if (n_tokens == 0) max_seqlen = 0;
    UNUM_CHECK_ARG(max_seqlen == 0 || (k_cache && v_cache && block_table), "null pointer argument");
    UNUM_CHECK_ARG(unum::aligned16(q) && unum::aligned16(k_cache) && unum::aligned16(v_cache) && unum::aligned16(out),
                   "q, k_cache, v_cache and out must be 16-byte aligned");
    UNUM_CHECK_ARG((q_sb | q_sh | k_st | k_sh | v_st | v_sh) % 8 == 0,
                   "strides of q, k_cache and v_cache must be multiples of 8 elements");
    UNUM_CHECK_ARG(B < 65536 && Hk < 65536 && B * Hk < ((int64_t)1 << 31), "too many sequences or kv heads");
    UNUM_CHECK_ARG(max_seqlen < ((int64_t)1 << 31), "max_seqlen must stay below 2^31");
    if (workspace_bytes < unum_paged_attention_workspace_size(B, Hq, Hk, D, max_seqlen, weights != nullptr) ||
        !workspace) {
        unum::set_error("workspace missing or too small (%lld bytes)", (long long)workspace_bytes);
        return UNUM_ERR_WORKSPACE;
    }
    Params p;
    p.q = q, p.kc = k_cache, p.vc = v_cache;
    p.q_sb = q_sb, p.q_sh = q_sh, p.k_st = k_st, p.k_sh = k_sh, p.v_st = v_st, p.v_sh = v_sh;
    p.table = block_table;
    p.lens = seqlens;
    p.bt_stride = bt_stride;
    p.n_tokens = n_tokens;
    p.max_len = max_seqlen;
    p.shift = 0;
    while (((int64_t)1 << p.shift) < page_size) ++p.shift;
    p.Hk = (int32_t)Hk;
    p.G = (int32_t)(Hq / Hk);
    p.c = softmax_scale * kLog2e;
    p.out = out;
    p.lse = lse;
    p.weights = weights;
    p.w_sb = w_sb;
    p.w_sh = w_sh;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == UNUM_DTYPE_BF16)
        return D == 128 ? launch<__nv_bfloat16, 128>(p, B, s) : launch<__nv_bfloat16, 64>(p, B, s);
    return D == 128 ? launch<__half, 128>(p, B, s) : launch<__half, 64>(p, B, s);
}
