// Attention of one new token for each sequence over its paged key-value cache.
//
// The reference has no dense attention over the cache; its get_block_table
// (src/unum_ops/sparse_kernel_extension/get_table_torch.py:29-44) fixes how a table maps positions to tokens.  For
// sequence b, query head h of kv head g = h / G and position p (page size P, a power of two):
//     token(p) = table[b, p / P] * P + p % P,   valid iff p < len_b and 0 <= token < n_tokens
//     s_p = scale * q[b,h] . k[token(p), g];   lse = log sum_p exp(s_p);   out = sum_p exp(s_p - lse) v[token(p), g]
//     weights[b,g,p] += sum over the group's heads of exp(s_p - lse)          (where they are gathered)
// A row without a valid position is 0 with lse = -inf.
//
// What bounds it: each key and value row is read once, 4 * D bytes a position and kv head, against 4 * D * G operations:
// at G = 16 and HBM's full rate 100 TFLOP/s, 6% of the tensor cores' rate.  So everything serves the loads:
//   - work is split over the length in units of 64 or 128 positions.  The units of all (sequence, kv head) items, in a
//     row, are dealt to the resident blocks in equal shares (two blocks an SM, one wave), so a batch of any lengths, one
//     long sequence or many short ones, loads every SM alike;
//   - a block's four warps take 16 positions at a time each.  A warp (a team of 2 or 4 warps where G > 16: one for each
//     16 heads) has a ring of its own in shared memory, filled by 16-byte asynchronous copies that gather rows by the
//     table, whose entries come into shared memory several steps before.  No block-wide barrier is in the loop, and the
//     copies run on across items;
//   - the products are m16n8k16 matrix instructions with the 16 heads as rows: scores and probabilities stay in
//     registers (the scores' layout is the layout that the second product wants), with the softmax's running maximum and
//     sum in 32 bits; the output accumulates in registers.  Tensor memory, with the keys as rows, would put a key in each
//     of its 128 lanes and so each maximum over keys across lanes, for a product that takes 6% of the tensor cores (with
//     the heads as rows it would not, but a tile has 64 rows at least: untried for groups of 64);
//   - where an item is cut, each block leaves its maximum, sum and output in the workspace and a second kernel joins them
//     in the order of the positions (the same bits each time).  It also turns the scores, left in the workspace in 32
//     bits, into weights: their sum over the group needs each head's final lse, and reading 4 * G bytes back costs less
//     than the key again;
//   - work so short that the second kernel would be a third of the time goes to clusters instead: one for each item, of
//     blocks with eight warps, which join their item through distributed shared memory.
// Measured (main kernel and join; a plain streaming read of the same bytes in brackets): 131072 positions of 2 x 128,
// G = 16: 25.3 + 6.8 us (24.8); 64 sequences of 4096 to 65536, 2.28 GB: 349 + 4.9 us, 6.5 TB/s (347); table entries
// read one step ahead only, 381 + 4.8; G = 32 over 134 MB 27.5 + 5.4, G = 64 43.6 + 8.7, where the matrix instructions'
// and the softmax's latency shows.
// Roundings: the probabilities go to the cache's type for the product with v (the sum l uses them unrounded), and the
// output once at the end.  The matrix instructions take no wider type beside the cache's; an output's error against 64
// bits, 1.7e-3 of its norm in bf16 and 2.0e-4 in fp16 with the last rounding alone, is 2.3e-3 and 2.6e-4 with both.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "sm100.cuh"

namespace {

using namespace unum::sm100;

constexpr int kBlocksPerSm = 2;
constexpr int kGrain = 2;            // units a block takes at least (1, 2 and 4 differ by less than 0.5 us)
constexpr int kMaxWorkers = 296;     // resident blocks, at most: two on each of 148 SMs
constexpr uint32_t kRingBytes = 96 * 1024;      // two blocks an SM
constexpr uint32_t kNearRingBytes = 192 * 1024;  // one: clusters that join their items have SMs to themselves
constexpr int kMaxG = 64;
constexpr int kMaxDevices = 64;
constexpr int kMaxUnit = 256;
constexpr int kMaxCluster = 16;
// Positions times head dim of a cluster's block, at most: where the clusters fill half of the SMs, and where they do not
// and dealing out would use the others.  Measured, cluster against dealt out and joined: one sequence of 217 positions
// 6.9 / 8.8 us, 1000 7.3 / 9.0, 4000 9.3 / 10.3, 8192 11.1 / 9.9; 64 of up to 500 10.8 / 13.9, 32 of up to 2000
// 14.3 / 17.3, 7 of up to 2501 with 8 kv heads of 64 9.6 / 11.2.
constexpr int kNearWork = 1024 * 128, kNearWorkAlone = 384 * 128;
constexpr int kJoinThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
    const uint8_t *q, *kc, *vc;
    int64_t q_sb, q_sh, k_sh, v_sh;  // bytes
    const int32_t *table, *lens;
    int64_t bt_stride, n_tokens;
    int32_t k_st, v_st;              // bytes
    int32_t max_len, shift, B, Hk, G, workers;
    float c;  // scale * log2(e)
    void *out;
    float *lse, *weights;
    int64_t w_sb, w_sh;
    // workspace
    int2 *span;          // [B * Hk]: first and last block of the item
    float *lse2;         // [B * Hk][16 * MT]: of items that one block holds, in base 2
    float2 *part_ml;     // [2 * workers][16 * MT]: maximum (base 2) and sum
    float4 *part_o;      // [2 * workers][MT][D / 8][32 lanes]
    float *scores;       // [B * Hk][G][score_ld], base 2
    int64_t score_ld;
};

// ---------------------------------------------------------------------------------------------- instructions
__device__ __forceinline__ uint64_t evict_first() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ uint64_t evict_last() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void st_hint(float *p, float x, float y, uint64_t policy) {
    asm volatile("st.global.L2::cache_hint.v2.f32 [%0], {%1, %2}, %3;" ::"l"(p), "f"(x), "f"(y), "l"(policy) : "memory");
}
__device__ __forceinline__ float4 ld_hint(const float *p, uint64_t policy) {
    float4 v;
    asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.f32 {%0, %1, %2, %3}, [%4], %5;"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p), "l"(policy) : "memory");
    return v;
}
// 16 zero bytes where `bytes` is 0
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes),
                 "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// kLift, kLag: see where the maximum is taken out
template <typename T> struct Num;
template <> struct Num<__nv_bfloat16> {
    static constexpr float kLift = 0.f, kUnlift = 1.f, kLag = 6.f;
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};
template <> struct Num<__half> {
    static constexpr float kLift = 12.f, kUnlift = 1.f / 4096, kLag = 3.f;  // kUnlift = 2^-kLift
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
};

// ---------------------------------------------------------------------------------------------- the order of the work
__device__ __forceinline__ int32_t length(const Params &p, int32_t b) {
    const int32_t n = p.lens[b];
    return n < 0 ? 0 : (n > p.max_len ? p.max_len : n);
}

// A place in the row of units: sequence, kv head, unit of the item.
template <int kUnit> struct Place {
    int32_t b, h, unit, units, len;
    __device__ __forceinline__ void set(const Params &p, int32_t b_) {
        b = b_;
        len = b < p.B ? length(p, b) : 0;
        units = (len + kUnit - 1) / kUnit;
    }
    __device__ __forceinline__ void next_item(const Params &p) {
        unit = 0;
        if (++h < p.Hk) return;
        h = 0;
        do set(p, b + 1);
        while (units == 0 && b < p.B);
    }
    __device__ __forceinline__ void next(const Params &p) {
        if (++unit == units) next_item(p);
    }
};

// Units before this thread's share of the sequences, and the total (over one kv head).  All threads call it.
template <int kN, int kUnit>
__device__ __forceinline__ int32_t scan_units(const Params &p, int32_t b0, int32_t b1, int32_t *warp_sums, int32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int32_t mine = 0;
    for (int32_t b = b0; b < b1; ++b) mine += (length(p, b) + kUnit - 1) / kUnit;
    int32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int32_t before = x - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kN; ++w) {
        if (w < warp) before += warp_sums[w];
        total += warp_sums[w];
    }
    return before;
}

// The units are dealt out in a row: the first `more` blocks have base + 1 of them, the others base.
struct Shares {
    int32_t base, more;
    __device__ __forceinline__ Shares() {}
    __device__ __forceinline__ Shares(int32_t total, int32_t workers) : base(total / workers), more(total % workers) {}
    __device__ __forceinline__ int32_t begin(int32_t w) const { return w * base + min(w, more); }
    __device__ __forceinline__ int32_t owner(int32_t u) const {
        const int32_t edge = more * (base + 1);
        return u < edge ? u / (base + 1) : more + (u - edge) / base;
    }
};

// MT = 16-head tiles of a group (1, 2 or 4): the warps of a team.  A team's step is 16 positions, or 32 where the ring has
// room for three such: the steps' barriers, maxima and copies cost half as much a position.  A unit, what is dealt out at
// a time, has a step for every team at least.
template <int D, int MT, bool kNear> struct Shape {
    static constexpr int kWarps = kNear ? 8 : 4, kThreads = kWarps * 32, kTeams = kWarps / MT;
    static constexpr int kStep = MT == 1 && D == 128 ? 16 : 32, kRow = D * 2;  // kRow in bytes
    static constexpr int kUnit = kTeams * kStep > 64 ? kTeams * kStep : 64;
    static constexpr int kSteps = kUnit / (kTeams * kStep);             // a team's steps in a unit
    static constexpr uint32_t kHalf = kStep * kRow, kSlot = 2 * kHalf;  // keys, values of a step
    static constexpr int kFit = (kNear ? kNearRingBytes : kRingBytes) / (kTeams * kSlot), kSlots = kFit > 8 ? 8 : kFit;
    // shared memory: the ring, what the teams leave for the first one (half of their columns at a time; a cluster's block
    // has the ring for that), the entries of the table that each warp has read ahead
    static constexpr int kBox = kNear ? 0 : (D / 16) * 32 * 16;
    static constexpr uint32_t kMergeAt = kTeams * kSlots * kSlot, kEntriesAt = kMergeAt + (kTeams - 1) * MT * kBox;
    static constexpr uint32_t kSmem = kEntriesAt + kWarps * kSlots * kStep * 4;
    static_assert(!kNear || kMergeAt >= (kWarps + MT) * (D / 8) * 32 * 16, "a cluster's block joins in the ring");
};

template <int D> __device__ __forceinline__ void write_empty(const Params &p, int64_t item, int threads) {
    uint32_t *op = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p.out) + item * p.G * D * 2);
    for (int i = threadIdx.x; i < p.G * D / 2; i += threads) op[i] = 0u;
    if (p.lse)
        for (int i = threadIdx.x; i < p.G; i += threads) p.lse[item * p.G + i] = -INFINITY;
}

// The weights that four positions from `pos` on gather from all heads of an item; z: the heads' lse in base 2.
__device__ __forceinline__ void gather4(const Params &p, int64_t item, const float *z, float *w, int32_t pos, int32_t end) {
    const float *sc = p.scores + item * p.G * p.score_ld + pos;
    // positions not held have a score of -inf: they gather nothing, even where the head's lse is NaN
    auto term = [](float s, float zh) { return s == -INFINITY || zh == -INFINITY ? 0.f : ex2(s - zh); };
    const uint64_t policy = evict_first();  // read once: what was kept for this makes room
    float old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (pos + i < end) old[i] = w[pos + i];
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int h = 0; h < p.G; ++h) {
        const float4 s = ld_hint(sc + h * p.score_ld, policy);
        const float zh = z[h];
        x.x += term(s.x, zh);
        x.y += term(s.y, zh);
        x.z += term(s.z, zh);
        x.w += term(s.w, zh);
    }
    const float add[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (pos + i < end) w[pos + i] = old[i] + add[i];
}

// What parts of one tile (rows r0 and r0 + 8 of a lane) add up to: maxima in base 2, sums, outputs.
struct Joined {
    float2 ml0, ml1;
    float4 o;
    __device__ __forceinline__ Joined()
        : ml0(make_float2(-INFINITY, 0.f)), ml1(make_float2(-INFINITY, 0.f)), o(make_float4(0.f, 0.f, 0.f, 0.f)) {}
    // Takes in n parts, four under way at once.  A loop and not unrolled: code that runs once waits for its instructions.
    template <typename Load> __device__ __forceinline__ void add(int n, const Load &load) {
#pragma unroll 1
        for (int i = 0; i < n; i += 4) {
            float2 a[4], b[4];
            float4 v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                a[e] = b[e] = make_float2(-INFINITY, 0.f);
                v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i + e < n) load(i + e, a[e], b[e], v[e]);
            }
            const float M0 = fmaxf(fmaxf(ml0.x, fmaxf(a[0].x, a[1].x)), fmaxf(a[2].x, a[3].x));
            const float M1 = fmaxf(fmaxf(ml1.x, fmaxf(b[0].x, b[1].x)), fmaxf(b[2].x, b[3].x));
            const float z0 = M0 == -INFINITY ? 0.f : M0, z1 = M1 == -INFINITY ? 0.f : M1;
            float f0 = ex2(ml0.x - z0), f1 = ex2(ml1.x - z1);
            ml0 = make_float2(M0, ml0.y * f0);
            ml1 = make_float2(M1, ml1.y * f1);
            o = make_float4(o.x * f0, o.y * f0, o.z * f1, o.w * f1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f0 = ex2(a[e].x - z0);
                f1 = ex2(b[e].x - z1);
                ml0.y += a[e].y * f0;
                ml1.y += b[e].y * f1;
                o.x += v[e].x * f0;
                o.y += v[e].y * f0;
                o.z += v[e].z * f1;
                o.w += v[e].w * f1;
            }
        }
    }
};

// What was taken out lies kLift below a maximum: back to it first, so that the two do not cancel.
template <typename T> __device__ __forceinline__ float lse2_of(float2 ml) {
    return ml.y != 0.f ? ml.x + Num<T>::kLift + log2f(ml.y * Num<T>::kUnlift) : -INFINITY;
}

// The end of an item that a cluster has: the block's warps leave their outputs, maxima and sums (ml: of rows r0 and
// r0 + 8) in shared memory and join them, tile by tile (8 columns of 16 heads); then each block joins some tiles of all
// blocks, and gathers the weights of its own positions.  All in the order of the warps and blocks: the same bits each time.
template <typename T, int D, int MT>
__device__ __forceinline__ void join_cluster(const Params &p, const float (&o)[D / 8][4], float2 ml0, float2 ml1, int64_t item,
                                             int32_t C, int32_t rank, int32_t u0, int32_t u1, int32_t len, uint8_t *smem) {
    using S = Shape<D, MT, true>;
    constexpr int kTiles = D / 8, kWarps = S::kWarps, kThreads = S::kThreads, kUnit = S::kUnit, kTeams = S::kTeams;
    __shared__ float2 warp_ml[kWarps][16], ml[16 * MT];
    __shared__ float z[16 * MT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r0 = lane >> 2;
    float4 *boxes = reinterpret_cast<float4 *>(smem);  // [kWarps][kTiles][32], where the ring was
    float4 *box = boxes + kWarps * kTiles * 32;        // [MT][kTiles][32]
    cp_wait<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTiles; ++i) boxes[(warp * kTiles + i) * 32 + lane] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    if ((lane & 3) == 0) {
        warp_ml[warp][r0] = ml0;
        warp_ml[warp][r0 + 8] = ml1;
    }
    __syncthreads();
#pragma unroll 1
    for (int t = warp; t < MT * kTiles; t += kWarps) {
        const int ht = t / kTiles, tile = t - ht * kTiles;
        Joined j;
        j.add(kTeams, [&](int w, float2 &a, float2 &b, float4 &v) {
            a = warp_ml[w * MT + ht][r0];
            b = warp_ml[w * MT + ht][r0 + 8];
            v = boxes[((w * MT + ht) * kTiles + tile) * 32 + lane];
        });
        box[t * 32 + lane] = j.o;
        if (tile == 0 && (lane & 3) == 0) {
            ml[ht * 16 + r0] = j.ml0;
            ml[ht * 16 + r0 + 8] = j.ml1;
        }
    }
    cluster_sync();
#pragma unroll 1
    for (int t = warp * C + rank; t < MT * kTiles; t += kWarps * C) {
        const int ht = t / kTiles, tile = t - ht * kTiles;
        Joined j;
        j.add(C, [&](int r, float2 &a, float2 &b, float4 &v) {
            a = ld_cluster_f32x2(peer_smem(&ml[ht * 16 + r0], r));
            b = ld_cluster_f32x2(peer_smem(&ml[ht * 16 + r0 + 8], r));
            v = ld_cluster_f32x4(peer_smem(&box[t * 32 + lane], r));
        });
        const float i0 = j.ml0.y != 0.f ? 1.f / j.ml0.y : 0.f, i1 = j.ml1.y != 0.f ? 1.f / j.ml1.y : 0.f;
        const int left = p.G - ht * 16;
        uint32_t *op = reinterpret_cast<uint32_t *>(
            static_cast<uint8_t *>(p.out) + ((item * p.G + ht * 16 + r0) * D + tile * 8 + (lane & 3) * 2) * 2);
        if (r0 < left) op[0] = Num<T>::pack(j.o.x * i0, j.o.y * i0);
        if (r0 + 8 < left) op[4 * D] = Num<T>::pack(j.o.z * i1, j.o.w * i1);
        if (p.lse && tile == 0 && (lane & 3) == 0) {
            float *l = p.lse + item * p.G + ht * 16 + r0;
            if (r0 < left) l[0] = lse2_of<T>(j.ml0) * kLn2;
            if (r0 + 8 < left) l[8] = lse2_of<T>(j.ml1) * kLn2;
        }
    }
    if (p.weights && tid < 16 * MT) {
        Joined j;
        j.add(C, [&](int r, float2 &a, float2 &, float4 &) { a = ld_cluster_f32x2(peer_smem(&ml[tid], r)); });
        z[tid] = lse2_of<T>(j.ml0);
    }
    cluster_arrive();
    if (p.weights) {
        __syncthreads();
        const int64_t b = item / p.Hk, g = item - b * p.Hk;
        const int32_t end = min(u1 * kUnit, len);
        for (int32_t pos = u0 * kUnit + 4 * tid; pos < end; pos += 4 * kThreads)
            gather4(p, item, z, p.weights + b * p.w_sb + g * p.w_sh, pos, end);
    }
    cluster_wait();  // no block leaves while another reads its shared memory
}

template <int MT> __device__ __forceinline__ void team_sync(int team) {
    __syncwarp();  // the barrier too is one that whole warps execute together
    if (MT > 1) asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(MT * 32) : "memory");
}

// kNear: a cluster has one item and joins it itself.
template <typename T, int D, int MT, bool kNear>
__global__ void __launch_bounds__(Shape<D, MT, kNear>::kThreads, kNear ? 1 : kBlocksPerSm)
    attend_kernel(const __grid_constant__ Params p) {
    using S = Shape<D, MT, kNear>;
    using N = Num<T>;
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads;
    constexpr int kTeams = S::kTeams, kStep = S::kStep, kSlots = S::kSlots, kRow = S::kRow, kUnit = S::kUnit;
    constexpr uint32_t kHalf = S::kHalf, kSlot = S::kSlot;
    constexpr int kLanes = kRow / 16, kRows = 32 / kLanes;  // lanes of a row, rows of one copy instruction
    constexpr int kCopies = kStep / kRows / MT;             // of each warp, for keys and for values
    static_assert(kCopies >= 1 && kSlots >= 3, "a step must give every warp a copy");
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint32_t held[kTeams][kSlots];            // which of a slot's positions are held
    __shared__ int2 ahead[kWarps][kSlots];               // of a step whose entries are read ahead: kv head, first position
    __shared__ int32_t warp_sums[kWarps], start[3];
    __shared__ float2 merge_ml[(kTeams > 1 ? kTeams - 1 : 1) * MT][16];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, team = warp / MT, ht = warp % MT;
    const uint32_t ring = smem_u32(smem) + team * (kSlots * kSlot);
    float4 *merge = reinterpret_cast<float4 *>(smem + S::kMergeAt);
    int32_t *entries = reinterpret_cast<int32_t *>(smem + S::kEntriesAt) + warp * (kSlots * kStep) + (lane & (kStep - 1));

    // Launched while the kernel before it may still run, and lets the one behind it do so.
    unum::wait_for_previous_kernel();
    const int32_t C = kNear ? cluster_nctarank() : 1, rank = kNear ? cluster_ctarank() : 0, me = blockIdx.x;
    int32_t u0, u1;
    Place<kUnit> in;  // where the entries are read
    Shares shares;
    if constexpr (kNear) {
        const int32_t item = me / C;
        in.b = item / p.Hk;
        in.h = item - in.b * p.Hk;
        in.set(p, in.b);
        if (in.len == 0) {
            if (rank == 0) write_empty<D>(p, item, kThreads);
            return;
        }
        shares = Shares(in.units, C);
        u0 = in.unit = shares.begin(rank);
        u1 = shares.begin(rank + 1);
    } else {
    // this block's share of the units
    const int32_t per = (p.B + kThreads - 1) / kThreads;
    const int32_t b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    int32_t total, before = scan_units<kWarps, kUnit>(p, b0, b1, warp_sums, total);
    before *= p.Hk;
    total *= p.Hk;
    const int32_t workers = min((total + kGrain - 1) / kGrain, p.workers);
    if (me >= workers) return;
    shares = Shares(total, workers);
    u0 = shares.begin(me);
    u1 = shares.begin(me + 1);
    for (int32_t b = b0; b < b1; ++b) {
        const int32_t n = (length(p, b) + kUnit - 1) / kUnit, mine = n * p.Hk;
        if (u0 >= before && u0 < before + mine) {
            const int32_t r = u0 - before;
            start[0] = b;
            start[1] = r / n;
            start[2] = r % n;
        }
        before += mine;
    }
    __syncthreads();
    in.set(p, start[0]);
    in.h = start[1];
    in.unit = start[2];
    }
    Place<kUnit> at = in;  // where the arithmetic is
    int32_t to_fetch = (u1 - u0) * S::kSteps;
    int in_k = 0;

    // Reads a step's table entries, lane % kStep for a position, on their way to shared memory: they are wanted
    // kSlots - 1 steps before the step's own turn, and come with the copies of the step that is waited for then.
    auto read_ahead = [&](uint32_t slot) {
        int32_t *to = entries + slot * kStep;
        if (to_fetch == 0) {
            *to = -1;
            return;
        }
        const int32_t pos0 = in.unit * kUnit + (team + kTeams * in_k) * kStep, pos = pos0 + (lane & (kStep - 1));
        if (pos >= in.len) *to = -1;
        else if (lane < kStep) cp_async4(smem_u32(to), p.table + in.b * p.bt_stride + (pos >> p.shift));
        if (lane == 0) ahead[warp][slot] = make_int2(in.h, pos0);
        --to_fetch;
        if (++in_k == S::kSteps) {
            in_k = 0;
            in.next(p);
        }
    };
    // A step's copies into its slot.  Rows of positions that are not held are zeroed: what their memory holds would reach
    // the output as 0 * NaN.  (Copies without that check where all 16 are held: the branch cost 8%.)
    constexpr uint32_t kAll = kStep == 32 ? 0xffffffffu : 0xffffu;
    const int copy_row = ht * kRows + lane / kLanes;
    const uint32_t copy_to = ring + copy_row * kRow;
    const uint32_t copy_chunk = lane % kLanes;
    // The cache passes through L2 once and makes room first, the scores stay until they are read (24 sequences of 2048 to
    // 32768 with weights: 101.6 us with the hint on the cache alone, 97.3 us with both).
    const uint64_t policy = evict_first(), keep = evict_last();
    auto issue = [&](uint32_t slot) {
        const int2 step = ahead[warp][slot];
        const int64_t page = entries[slot * kStep];
        const int64_t token = (page << p.shift) + ((step.y + (lane & (kStep - 1))) & ((1 << p.shift) - 1));
        const int32_t tok = page >= 0 && token < p.n_tokens ? (int32_t)token : -1;
        const uint32_t mask = __ballot_sync(0xffffffffu, tok >= 0) & kAll;
        if (ht == 0 && lane == 0) held[team][slot] = mask;
        if (mask) {
            const uint8_t *kb = p.kc + step.x * p.k_sh + copy_chunk * 16;
            const uint8_t *vb = p.vc + step.x * p.v_sh + copy_chunk * 16;
            const uint32_t to = copy_to + slot * kSlot;
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int row = i * MT * kRows + copy_row;
                const int32_t t = __shfl_sync(0xffffffffu, tok, row);
                const uint32_t dst = to + i * MT * kRows * kRow + ((copy_chunk ^ (row & 7)) << 4);
                const int64_t o = t < 0 ? 0 : t;
                cp_async16(dst, kb + o * p.k_st, t < 0 ? 0u : 16u, policy);
                cp_async16(dst + kHalf, vb + o * p.v_st, t < 0 ? 0u : 16u, policy);
            }
        }
        read_ahead(slot == 0 ? kSlots - 1 : slot - 1);
        cp_commit();
    };

#pragma unroll 1
    for (int s = 0; s < kSlots - 1; ++s) read_ahead(s);
    cp_commit();
    cp_wait<0>();
    __syncwarp();
#pragma unroll 1
    for (int s = 0; s < kSlots - 1; ++s) issue(s);

    uint32_t slot = 0;
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    // rows and swizzled 16-byte chunks of the matrices that this lane addresses; chunk 2 kk + e is that xor 2 kk
    const int k_row = (lane & 7) + ((lane >> 4) << 3), v_row = lane & 15;
    const uint32_t k_at = k_row * kRow + ((((lane >> 3) & 1) ^ (k_row & 7)) << 4);
    const uint32_t v_at = v_row * kRow + (((lane >> 4) ^ (v_row & 7)) << 4);
    int32_t u = u0;
    while (kNear || u < u1) {  // kNear: once, also without a unit
        // one item's units in this block
        const int32_t seg_end = kNear ? u1 : min(u + (at.units - at.unit), u1);
        const bool from_start = at.unit == 0, to_end = u + (at.units - at.unit) == seg_end;
        const int64_t item = (int64_t)at.b * p.Hk + at.h;
        const int32_t item_u0 = u - at.unit;
        uint32_t qa[D / 16][4];
        {
            const uint8_t *qb = p.q + at.b * p.q_sb + (int64_t)(at.h * p.G + ht * 16) * p.q_sh + c0 * 2;
            const int left = p.G - ht * 16;
            const uint8_t *q0 = qb + r0 * p.q_sh, *q1 = qb + (r0 + 8) * p.q_sh;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                qa[k][0] = r0 < left ? *reinterpret_cast<const uint32_t *>(q0 + k * 32) : 0u;
                qa[k][1] = r0 + 8 < left ? *reinterpret_cast<const uint32_t *>(q1 + k * 32) : 0u;
                qa[k][2] = r0 < left ? *reinterpret_cast<const uint32_t *>(q0 + k * 32 + 16) : 0u;
                qa[k][3] = r0 + 8 < left ? *reinterpret_cast<const uint32_t *>(q1 + k * 32 + 16) : 0u;
            }
        }
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        float *sc = p.scores + (item * p.G + ht * 16 + r0) * p.score_ld + c0;

        for (; u < seg_end; ++u, ++at.unit) {
#pragma unroll 1
            for (int k = 0; k < S::kSteps; ++k) {
                cp_wait<kSlots - 2>();
                team_sync<MT>(team);  // the slot is filled, and nobody reads the one before it any more
                issue(slot == 0 ? kSlots - 1 : slot - 1);
                const uint32_t mask = held[team][slot];
                const uint32_t kb = ring + slot * kSlot + k_at, vb = ring + slot * kSlot + kHalf + v_at;
                slot = slot + 1 == kSlots ? 0 : slot + 1;
                if (mask == 0 && !p.weights) continue;
                float s[kStep / 8][4];
#pragma unroll
                for (int t = 0; t < kStep / 8; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
                if (kStep == 16 && mask) {
                    // two chains of products for each 8 positions: half the latency, half the roundings in a row
                    float e[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk += 2) {
                        uint32_t f[4], g[4];
                        ldsm4(f, kb ^ (kk << 5));
                        ldsm4(g, kb ^ ((kk + 1) << 5));
                        Num<T>::mma(s[0], qa[kk], f[0], f[1]);
                        Num<T>::mma(s[1], qa[kk], f[2], f[3]);
                        Num<T>::mma(e[0], qa[kk + 1], g[0], g[1]);
                        Num<T>::mma(e[1], qa[kk + 1], g[2], g[3]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] += e[i >> 2][i & 3];
                } else if (mask) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                        for (int t = 0; t < kStep / 16; ++t) {
                            uint32_t f[4];
                            ldsm4(f, (kb ^ (kk << 5)) + t * 16 * kRow);
                            Num<T>::mma(s[2 * t], qa[kk], f[0], f[1]);
                            Num<T>::mma(s[2 * t + 1], qa[kk], f[2], f[3]);
                        }
                }
#pragma unroll
                for (int t = 0; t < kStep / 8; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][e] *= p.c;
                if (mask != kAll) {
                    const uint32_t mine = mask >> c0;
#pragma unroll
                    for (int t = 0; t < kStep / 8; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!((mine >> (8 * t + (e & 1))) & 1u)) s[t][e] = -INFINITY;
                }
                if (p.weights) {
                    const int64_t pos = (int64_t)at.unit * kUnit + (team + kTeams * k) * kStep;
                    if (pos < at.len) {
#pragma unroll
                        for (int t = 0; t < kStep / 8; ++t) {
                            if (ht * 16 + r0 < p.G)
                                st_hint(sc + pos + 8 * t, s[t][0], s[t][1], keep);
                            if (ht * 16 + r0 + 8 < p.G)
                                st_hint(sc + 8 * p.score_ld + pos + 8 * t, s[t][2], s[t][3], keep);
                        }
                    }
                    if (mask == 0) continue;
                }
                float x0 = fmaxf(s[0][0], s[0][1]), x1 = fmaxf(s[0][2], s[0][3]);
#pragma unroll
                for (int t = 1; t < kStep / 8; ++t) {
                    x0 = fmaxf(x0, fmaxf(s[t][0], s[t][1]));
                    x1 = fmaxf(x1, fmaxf(s[t][2], s[t][3]));
                }
#pragma unroll
                for (int i = 1; i <= 2; i <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, i));
                    x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, i));
                }
                // What is taken out lies kLift below a maximum, so that probabilities come to 2^kLift: fp16 has all its
                // bits from 2^-14 on only, and would lose those of keys far below one that outshines them.  And the maximum
                // may stay behind the true one by up to kLag: the output is rescaled that much more rarely.  Together they
                // leave probabilities up to 2^15 in fp16, whose largest is just below 2^16.  The difference is what is
                // looked at, and a maximum so large that its last place passes kLift is taken out as it is: neither limit
                // holds after rounding otherwise.
                if (__any_sync(0xffffffffu, x0 - m0 > N::kLift + N::kLag || x1 - m1 > N::kLift + N::kLag)) {
                    x0 = fmaxf(x0 - (x0 - N::kLift) <= N::kLift ? x0 - N::kLift : x0, m0);
                    x1 = fmaxf(x1 - (x1 - N::kLift) <= N::kLift ? x1 - N::kLift : x1, m1);
                    const float a0 = x0 == -INFINITY ? 1.f : ex2(m0 - x0), a1 = x1 == -INFINITY ? 1.f : ex2(m1 - x1);
                    m0 = x0;
                    m1 = x1;
                    l0 *= a0;
                    l1 *= a1;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        o[i][0] *= a0;
                        o[i][1] *= a0;
                        o[i][2] *= a1;
                        o[i][3] *= a1;
                    }
                }
                const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
                for (int t = 0; t < kStep / 8; ++t) {
                    s[t][0] = ex2(s[t][0] - z0);
                    s[t][1] = ex2(s[t][1] - z0);
                    s[t][2] = ex2(s[t][2] - z1);
                    s[t][3] = ex2(s[t][3] - z1);
                    l0 += s[t][0] + s[t][1];
                    l1 += s[t][2] + s[t][3];
                }
#pragma unroll
                for (int t = 0; t < kStep / 16; ++t) {
                    const uint32_t a[4] = {
                        Num<T>::pack(s[2 * t][0], s[2 * t][1]), Num<T>::pack(s[2 * t][2], s[2 * t][3]),
                        Num<T>::pack(s[2 * t + 1][0], s[2 * t + 1][1]), Num<T>::pack(s[2 * t + 1][2], s[2 * t + 1][3])};
#pragma unroll
                    for (int nn = 0; nn < D / 16; ++nn) {
                        uint32_t f[4];
                        ldsm4t(f, (vb ^ (nn << 5)) + t * 16 * kRow);
                        Num<T>::mma(o[2 * nn], a, f[0], f[1]);
                        Num<T>::mma(o[2 * nn + 1], a, f[2], f[3]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 1; i <= 2; i <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, i);
            l1 += __shfl_xor_sync(0xffffffffu, l1, i);
        }
        if constexpr (kNear) {
            join_cluster<T, D, MT>(p, o, make_float2(m0, l0), make_float2(m1, l1), item, C, rank, u0, u1, at.len, smem);
            return;
        }
        // the first team takes in what the others leave, half of the columns at a time
        if constexpr (!kNear && kTeams > 1) {
            if (team > 0 && (lane & 3) == 0) {
                merge_ml[warp - MT][r0] = make_float2(m0, l0);
                merge_ml[warp - MT][r0 + 8] = make_float2(m1, l1);
            }
            float f0[kTeams], f1[kTeams];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (team > 0) {
                    float4 *box = merge + (warp - MT) * (D / 16) * 32 + lane;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const float(&x)[4] = o[half * (D / 16) + i];
                        box[i * 32] = make_float4(x[0], x[1], x[2], x[3]);
                    }
                }
                __syncthreads();
                if (team == 0) {
                    if (half == 0) {
                        float n0 = m0, n1 = m1;
#pragma unroll
                        for (int w = 1; w < kTeams; ++w) {
                            n0 = fmaxf(n0, merge_ml[(w - 1) * MT + ht][r0].x);
                            n1 = fmaxf(n1, merge_ml[(w - 1) * MT + ht][r0 + 8].x);
                        }
                        const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
                        f0[0] = ex2(m0 - z0);
                        f1[0] = ex2(m1 - z1);
                        m0 = n0;
                        m1 = n1;
                        l0 *= f0[0];
                        l1 *= f1[0];
#pragma unroll
                        for (int w = 1; w < kTeams; ++w) {
                            const float2 y0 = merge_ml[(w - 1) * MT + ht][r0], y1 = merge_ml[(w - 1) * MT + ht][r0 + 8];
                            f0[w] = ex2(y0.x - z0);
                            f1[w] = ex2(y1.x - z1);
                            l0 += y0.y * f0[w];
                            l1 += y1.y * f1[w];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        float(&x)[4] = o[half * (D / 16) + i];
                        x[0] *= f0[0];
                        x[1] *= f0[0];
                        x[2] *= f1[0];
                        x[3] *= f1[0];
#pragma unroll
                        for (int w = 1; w < kTeams; ++w) {
                            const float4 y = merge[(((w - 1) * MT + ht) * (D / 16) + i) * 32 + lane];
                            x[0] += y.x * f0[w];
                            x[1] += y.y * f0[w];
                            x[2] += y.z * f1[w];
                            x[3] += y.w * f1[w];
                        }
                    }
                }
                __syncthreads();
            }
        }
        if (team == 0) {
            if (from_start && to_end) {  // the whole item
                const float i0 = l0 != 0.f ? 1.f / l0 : 0.f, i1 = l1 != 0.f ? 1.f / l1 : 0.f;
                const float z0 = lse2_of<T>(make_float2(m0, l0)), z1 = lse2_of<T>(make_float2(m1, l1));
                const int left = p.G - ht * 16;
                uint32_t *op = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p.out) +
                                                            ((item * p.G + ht * 16 + r0) * D + c0) * 2);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    if (r0 < left) op[i * 4] = Num<T>::pack(o[i][0] * i0, o[i][1] * i0);
                    if (r0 + 8 < left) op[i * 4 + 4 * D] = Num<T>::pack(o[i][2] * i1, o[i][3] * i1);
                }
                if ((lane & 3) == 0) {
                    float *z = p.lse2 + item * (16 * MT) + ht * 16 + r0;
                    z[0] = z0;
                    z[8] = z1;
                    if (p.lse) {
                        float *l = p.lse + item * p.G + ht * 16 + r0;
                        if (r0 < left) l[0] = z0 * kLn2;
                        if (r0 + 8 < left) l[8] = z1 * kLn2;
                    }
                }
            } else {
                // an item's first part is its block's last work, every other part its block's first
                const int64_t spot = 2 * me + (from_start ? 1 : 0);
                float4 *po = p.part_o + (spot * MT + ht) * (D / 8) * 32 + lane;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) po[i * 32] = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
                if ((lane & 3) == 0) {
                    float2 *ml = p.part_ml + spot * (16 * MT) + ht * 16 + r0;
                    ml[0] = make_float2(m0, l0);
                    ml[8] = make_float2(m1, l1);
                }
            }
            if (to_end && warp == 0 && lane == 0) {
                p.span[item] = make_int2(shares.owner(item_u0), me);
            }
        }
        at.unit = at.units - 1;
        at.next(p);
    }
    cp_wait<0>();
}

// Joins the parts of items that were cut (blocks y < splits: each has `tiles` of the output's 8-column tiles of one
// 16-head tile, and slices = 16 / tiles warps share a tile's parts), and gathers weights (the other blocks y).  Blocks
// x: items.  All of it is latency: every load of a thread that another does not need first is under way at once.
template <typename T, int D, int MT>
__global__ void __launch_bounds__(kJoinThreads, 2) join_kernel(const __grid_constant__ Params p, int32_t tiles, int32_t splits) {
    constexpr int kJoinWarps = kJoinThreads / 32, kBatch = 5;
    __shared__ float2 ml[kMaxWorkers][17];  // of each part and head: maximum and sum.  17: banks
    __shared__ float4 sums[kJoinWarps][32];
    __shared__ __align__(16) float z[kMaxG];
    unum::wait_for_previous_kernel();
    const int32_t item = blockIdx.x, b = item / p.Hk, g = item - b * p.Hk;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t len = length(p, b);
    const bool join = (int)blockIdx.y < splits;
    const int2 sp = __ldcg(&p.span[item]);
    if (len == 0) {
        if (blockIdx.y == 0) write_empty<D>(p, item, kJoinThreads);
        return;
    }
    const int32_t parts = sp.y - sp.x + 1;
    if (join && parts == 1) return;
    auto spot = [&](int32_t i) { return 2 * (int64_t)(sp.x + i) + (i == 0 ? 1 : 0); };
    // M and L of each head of a tile, one warp a head; ml becomes 2^(m - M) / L of each part and head
    auto stats = [&](int ht) {
        for (int32_t i = tid; i < parts * 16; i += kJoinThreads)
            ml[i >> 4][i & 15] = __ldcg(&p.part_ml[spot(i >> 4) * (16 * MT) + ht * 16 + (i & 15)]);
        __syncthreads();
        float M = -INFINITY, L = 0.f;
        for (int32_t i = lane; i < parts; i += 32) M = fmaxf(M, ml[i][warp].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float base = M == -INFINITY ? 0.f : M;
        for (int32_t i = lane; i < parts; i += 32) {
            const float2 v = ml[i][warp];
            const float f = ex2(v.x - base);
            L += v.y * f;
            ml[i][warp].x = f;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const float inv = L != 0.f ? 1.f / L : 0.f;
        for (int32_t i = lane; i < parts; i += 32) ml[i][warp].x *= inv;
        const float lse2 = lse2_of<T>(make_float2(M, L));
        if (lane == 0) z[ht * 16 + warp] = lse2;
        __syncthreads();
        return lse2;
    };
    if (join) {
        const int slices = kJoinWarps / tiles, per_ht = D / 8 / tiles;
        const int ht = blockIdx.y / per_ht, tile = blockIdx.y % per_ht * tiles + warp / slices;
        const float4 *src = p.part_o + (int64_t)(ht * (D / 8) + tile) * 32 + lane;
        const int32_t i0 = warp % slices;
        float4 v[kBatch];
        auto load = [&](int32_t i) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (i + j * slices < parts) v[j] = __ldcg(src + spot(i + j * slices) * (MT * (D / 8) * 32));
        };
        load(i0);  // while M and L are found
        const float lse2 = stats(ht);
        if (p.lse && blockIdx.y % per_ht == 0 && lane == 0 && ht * 16 + warp < p.G)
            p.lse[(int64_t)item * p.G + ht * 16 + warp] = lse2 * kLn2;
        const int r0 = lane >> 2;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int32_t i = i0; i < parts; i += kBatch * slices) {
            if (i != i0) load(i);
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (i + j * slices < parts) {
                    const float f0 = ml[i + j * slices][r0].x, f1 = ml[i + j * slices][r0 + 8].x;
                    acc.x += v[j].x * f0;
                    acc.y += v[j].y * f0;
                    acc.z += v[j].z * f1;
                    acc.w += v[j].w * f1;
                }
        }
        if (slices > 1) {
            sums[warp][lane] = acc;
            __syncthreads();
            if (i0) return;
            for (int i = 1; i < slices; ++i) {
                const float4 y = sums[warp + i][lane];
                acc.x += y.x;
                acc.y += y.y;
                acc.z += y.z;
                acc.w += y.w;
            }
        }
        const int left = p.G - ht * 16;
        uint32_t *op = reinterpret_cast<uint32_t *>(
            static_cast<uint8_t *>(p.out) + (((int64_t)item * p.G + ht * 16 + r0) * D + tile * 8 + (lane & 3) * 2) * 2);
        if (r0 < left) op[0] = Num<T>::pack(acc.x, acc.y);
        if (r0 + 8 < left) op[4 * D] = Num<T>::pack(acc.z, acc.w);
        return;
    }
    // weights: four positions a thread
    if (parts == 1) {
        if (tid < p.G) z[tid] = __ldcg(&p.lse2[(int64_t)item * (16 * MT) + tid]);
    } else {
        for (int ht = 0; ht < MT; ++ht) stats(ht);
    }
    __syncthreads();
    const int32_t n_blocks = gridDim.y - splits, mine = blockIdx.y - splits;
    for (int64_t pos = 4 * ((int64_t)mine * kJoinThreads + tid); pos < len; pos += 4 * (int64_t)n_blocks * kJoinThreads)
        gather4(p, item, z, p.weights + b * p.w_sb + g * p.w_sh, (int32_t)pos, len);
}

int64_t workers_of_device() {
    const int64_t n = (int64_t)unum::sm_count() * kBlocksPerSm;
    return n < kMaxWorkers ? n : kMaxWorkers;
}

int head_tiles(int64_t G) { return G <= 16 ? 1 : (G <= 32 ? 2 : 4); }

// The workspace's parts, in order; each a multiple of 16 bytes.
struct Layout {
    size_t span, lse2, part_ml, part_o, scores, bytes;
    int64_t score_ld;
};

Layout layout_of(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t max_len, bool gather) {
    const int64_t W = workers_of_device(), rows = 16 * head_tiles(Hq / Hk), items = B * Hk;
    Layout l;
    size_t at = 0;
    auto take = [&](int64_t bytes) {
        const size_t o = at;
        at += ((size_t)bytes + 15) / 16 * 16;
        return o;
    };
    l.part_o = take(2 * W * rows * D * 4);
    l.part_ml = take(2 * W * rows * 8);
    l.span = take(items * 8);
    l.lse2 = take(items * rows * 4);
    l.score_ld = (max_len + kMaxUnit - 1) / kMaxUnit * kMaxUnit;
    l.scores = take(gather ? items * (Hq / Hk) * l.score_ld * 4 : 0);
    l.bytes = at;
    return l;
}

// Clusters of 2^i blocks of a kernel that are resident at once on the current device.
int active_clusters(const void *kernel, cudaLaunchConfig_t &cfg, std::atomic<int32_t> (&known)[kMaxDevices][5], int i) {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices) return 0;
    if (const int have = known[dev][i].load(std::memory_order_relaxed)) return have - 1;
    cfg.attrs[0].val.clusterDim.x = 1u << i;
    cfg.gridDim = dim3(1u << i);
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    known[dev][i].store(n + 1, std::memory_order_relaxed);
    return n;
}

template <typename T, int D, int MT> int launch(const Params &p, cudaStream_t s) {
    const int64_t items = (int64_t)p.B * p.Hk;
    {
        // A cluster that has one item joins it itself, without a second kernel, but its blocks idle where other sequences
        // are longer: it pays where every item at its longest is short work for its blocks, and all are resident at once.
        using S = Shape<D, MT, true>;
        auto *kernel = attend_kernel<T, D, MT, true>;
        static std::atomic<int32_t> known[kMaxDevices][5];
        UNUM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::kSmem));
        UNUM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t cfg = {};
        cfg.blockDim = dim3(S::kThreads);
        cfg.dynamicSmemBytes = S::kSmem;
        cfg.stream = s;
        cudaLaunchAttribute attr[2] = {};
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1] = unum::behind_previous_kernel();
        cfg.attrs = attr;
        cfg.numAttrs = 1;  // what the occupancy takes
        const int64_t units = ((int64_t)p.max_len + S::kUnit - 1) / S::kUnit;
        int i = 0;
        while ((2 << i) <= kMaxCluster && (1 << i) < units &&
               items <= active_clusters((const void *)kernel, cfg, known, i + 1))
            ++i;
        const int64_t C = 1 << i;
        if (items <= active_clusters((const void *)kernel, cfg, known, i) &&
            (units + C - 1) / C * S::kUnit * D <= (2 * items * C >= unum::sm_count() ? kNearWork : kNearWorkAlone)) {
            cfg.gridDim = dim3((unsigned)(items * C));
            attr[0].val.clusterDim.x = (unsigned)C;
            cfg.numAttrs = 2;
            UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
            return unum::check_launch("attend_kernel");
        }
    }
    auto *kernel = attend_kernel<T, D, MT, false>;
    constexpr uint32_t smem = Shape<D, MT, false>::kSmem;
    UNUM_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchAttribute attr = unum::behind_previous_kernel();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.workers);
    cfg.blockDim = dim3(Shape<D, MT, false>::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    // A long item is cut into about workers / items parts, and then a block of the second kernel has one tile's columns
    // and 16 warps on its parts; where items are many they have a few parts each, and a block has the whole row.
    int tiles = D / 8;
    while (tiles > 1 && 16 / tiles * 4 * items < p.workers) tiles /= 2;
    const int splits = MT * (D / 8) / tiles;
    int64_t gather = 0;
    if (p.weights) {
        gather = (4 * (int64_t)p.workers + items - 1) / items;
        const int64_t most = ((int64_t)p.max_len + 4 * kJoinThreads - 1) / (4 * kJoinThreads);
        if (gather > most) gather = most;
    }
    cfg.gridDim = dim3((unsigned)items, (unsigned)(splits + gather));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    UNUM_CHECK_CUDA(cudaLaunchKernelEx(&cfg, join_kernel<T, D, MT>, p, (int32_t)tiles, (int32_t)splits));
    return unum::check_launch("join_kernel");
}

template <typename T> int launch_for(const Params &p, int64_t D, cudaStream_t s) {
    const int mt = head_tiles(p.G);
    if (D == 128) return mt == 1 ? launch<T, 128, 1>(p, s) : mt == 2 ? launch<T, 128, 2>(p, s) : launch<T, 128, 4>(p, s);
    return mt == 1 ? launch<T, 64, 1>(p, s) : mt == 2 ? launch<T, 64, 2>(p, s) : launch<T, 64, 4>(p, s);
}

}  // namespace

extern "C" size_t unum_paged_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hk, int64_t D, int64_t max_seqlen,
                                                      int gather_weights) {
    if (B < 0 || Hq <= 0 || Hk <= 0 || Hq < Hk || D <= 0 || max_seqlen < 0) return 0;
    return layout_of(B, Hq, Hk, D, max_seqlen, gather_weights != 0).bytes;
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
    UNUM_CHECK_ARG(k_st >= 0 && k_st < (1 << 30) && v_st >= 0 && v_st < (1 << 30),
                   "token strides of k_cache and v_cache must be below 2^30 elements");
    UNUM_CHECK_ARG(Hk < 65536 && B < ((int64_t)1 << 31) / Hk &&
                       B * Hk < ((int64_t)1 << 31) / (max_seqlen / 64 + 2),
                   "too many sequences, kv heads or positions");
    UNUM_CHECK_ARG(max_seqlen <= ((int64_t)1 << 31) - 2 * kMaxUnit && n_tokens < ((int64_t)1 << 31),
                   "max_seqlen and n_tokens must stay below 2^31");
    const Layout l = layout_of(B, Hq, Hk, D, max_seqlen, weights != nullptr);
    if (workspace_bytes < l.bytes || !workspace || !unum::aligned16(workspace)) {
        unum::set_error("workspace missing, misaligned or too small (%lld bytes; %lld needed)", (long long)workspace_bytes,
                        (long long)l.bytes);
        return UNUM_ERR_WORKSPACE;
    }
    Params p;
    p.q = (const uint8_t *)q, p.kc = (const uint8_t *)k_cache, p.vc = (const uint8_t *)v_cache;
    p.q_sb = 2 * q_sb, p.q_sh = 2 * q_sh, p.k_sh = 2 * k_sh, p.v_sh = 2 * v_sh;
    p.k_st = (int32_t)(2 * k_st), p.v_st = (int32_t)(2 * v_st);
    p.table = block_table;
    p.lens = seqlens;
    p.bt_stride = bt_stride;
    p.n_tokens = n_tokens;
    p.max_len = (int32_t)max_seqlen;
    p.shift = 0;
    while (((int64_t)1 << p.shift) < page_size) ++p.shift;
    p.B = (int32_t)B;
    p.Hk = (int32_t)Hk;
    p.G = (int32_t)(Hq / Hk);
    // no more blocks than the lengths can give units to
    const int64_t most = B * Hk * ((max_seqlen + 63) / 64), W = workers_of_device();
    p.workers = (int32_t)(most < 1 ? 1 : (most < W ? most : W));
    p.c = softmax_scale * kLog2e;
    p.out = out;
    p.lse = lse;
    p.weights = weights;
    p.w_sb = w_sb;
    p.w_sh = w_sh;
    uint8_t *ws = (uint8_t *)workspace;
    p.span = (int2 *)(ws + l.span);
    p.lse2 = (float *)(ws + l.lse2);
    p.part_ml = (float2 *)(ws + l.part_ml);
    p.part_o = (float4 *)(ws + l.part_o);
    p.scores = (float *)(ws + l.scores);
    p.score_ld = l.score_ld;
    cudaStream_t s = (cudaStream_t)stream;
    return dtype == UNUM_DTYPE_BF16 ? launch_for<__nv_bfloat16>(p, D, s) : launch_for<__half>(p, D, s);
}
