// Log-probability of one token per row of logits, and the clipped policy loss with a KL term on it, forward and backward in one pass.
// With S = sum over j != y of exp(x[j]) the log-probability of token y is lp = -log(1 + S / exp(x[y])), and
//   ratio = exp(lp - old),  gain = min(ratio * A, clip(ratio, 1 - low, 1 + high) * A),  kl = exp(ref - lp) - (ref - lp) - 1
//   row_loss = weight * (kl_coef * kl - gain)
//   d_logits[j] = slope * ([j = y] - p[j]),  slope = weight * (kl_coef * (1 - exp(ref - lp)) - (ratio * A where gain is not the clipped one))
// Keeping y out of S keeps lp and 1 - p[y] exact to rounding however likely y is. Exponentials and sums are fp32, a row's few scalars 64-bit, so
// that a ratio next to its clip is on the right side. An exponential is 2^((x[j] - m) log2 e), m a running maximum that is one of the logits: the
// difference is exact next to the maximum and overflows to nothing but -inf, so that finite logits of any size, a row that is masked as a whole by
// the type's lowest value among them, have the weights that the formula gives them. One fused x[j] log2 e - m log2 e would overflow there, and be
// off by the rounding of m log2 e.
//
// Bound by HBM: logits are read once and gradients written once. A row of a 151 936-word vocabulary is 608 KB, so a thread-block cluster
// holds it in its shared memory between the sum and the gradient: each block one slice, fetched by bulk copies in pieces of 16 KB that
// are summed as they land; the blocks exchange (maximum, sum, x[y]) through distributed shared memory. Slices of 76 KB leave three
// blocks an SM, so that one row's copies run under another's arithmetic and stores (2 048 rows of 151 936 fp32, a quarter of them masked: 428 us,
// 5.1 TB/s; blocks of 512 threads 434 us, and two of them an SM with slices of 108 KB 460 us; clusters of 14 with slices of 44 KB 454 us).
#include "launch.h"
#include "pair.cuh"
#include "ptx.cuh"
#include "train.h"
#include <algorithm>
#include <cfloat>

namespace tffn {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPiece = 16384;              // bytes of a bulk copy
constexpr int kMaxSlice = 216 * 1024;      // bytes of a row that one block can hold
constexpr int kPerSm = 3, kSharedSlice = (228 * 1024 / kPerSm - 1024 - 600) / 16 * 16;  // the same with three blocks an SM
constexpr int kMaxBlocks = 8;              // blocks of a cluster
constexpr int kMaxPieces = (kMaxSlice + kPiece - 1) / kPiece;
constexpr int kHead = 256;                 // barriers and the blocks' partial results, in front of the slice

// 2^x, x up to 0, on the FMA pipe: x = n + f with |f| <= 1/2, 2^f by a polynomial of degree 6 fitted for the least largest relative error (Remez
// exchange; 1.6e-8 with coefficients rounded to fp32), times 2^n; off by 7.9e-8 at most and not to one side. For the factors by which partial sums are joined: those of the exponential
// unit are off to one side, ten of them in a row by 2.5e-7 (mean error of a log-probability over 32 768 words; with these 2e-8), and a KL term of a hundredth
// multiplies that by fourteen. The single terms' errors average out; polynomials for them as well cost 18% of the time for nothing measurable.
// 0 below -126, NaN of NaN.
__device__ __forceinline__ float exp2_exact(float x) {
    const float big = 12582912.f + 127.f;  // 1.5 * 2^23: adding it rounds to an integer, which is then the low bits; 127: the exponent of 1
    const float t = x + big, f = x - (t - big);
    float y = 0.0001534581242594868f;
    y = fmaf(y, f, 0.0013399930903688073f);
    y = fmaf(y, f, 0.009618489071726799f);
    y = fmaf(y, f, 0.05550328642129898f);
    y = fmaf(y, f, 0.24022646248340607f);
    y = fmaf(y, f, 0.6931471824645996f);
    y = fmaf(y, f, 1.f);
    return x < -126.f ? 0.f : y * __int_as_float(__float_as_int(t) << 23);
}

// running maximum, and sum of exp(x - maximum)
struct Lse {
    float m = -FLT_MAX, s = 0.f;
    __device__ __forceinline__ void join(float m2, float s2) {
        const float top = fmaxf(m, m2);
        s = s * exp2_exact((m - top) * kLog2e) + s2 * exp2_exact((m2 - top) * kLog2e);
        m = top;
    }
};

template <typename T>
struct Pack;  // 16 bytes of logits
template <>
struct Pack<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(uint4 v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <>
struct Pack<bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(uint4 v, float (&f)[8]) {
        f[0] = bf16_lo(v.x);
        f[1] = bf16_hi(v.x);
        f[2] = bf16_lo(v.y);
        f[3] = bf16_hi(v.y);
        f[4] = bf16_lo(v.z);
        f[5] = bf16_hi(v.z);
        f[6] = bf16_lo(v.w);
        f[7] = bf16_hi(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *(const uint32_t*)&h;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// exp(f[i] - m), two differences and two products an instruction (log-probabilities of 1 024 x 151 936 bf16: 64 us, one at a time 70)
template <int N>
__device__ __forceinline__ void weights(float (&f)[N], float m) {
    if constexpr (N % 2 == 0) {
        const F2 m2 = f2(-m, -m), k2 = f2(kLog2e, kLog2e);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            split2(mul2(add2(f2(f[i], f[i + 1]), m2), k2), f[i], f[i + 1]);
            f[i] = exp2_fast(f[i]);
            f[i + 1] = exp2_fast(f[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = exp2_fast((f[i] - m) * kLog2e);
    }
}

// N values at indices first ..; the one at index `skip` is left out
template <int N>
__device__ __forceinline__ void take(Lse& l, const float (&f)[N], int first, int skip) {
    float t[N], top = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        t[i] = f[i];
        if ((unsigned)(skip - first) < (unsigned)N && first + i == skip) t[i] = -INFINITY;
        top = fmaxf(top, t[i]);
    }
    if (top > l.m) {
        l.s *= exp2_fast((l.m - top) * kLog2e);
        l.m = top;
    }
    weights(t, l.m);
#pragma unroll
    for (int i = 0; i < N; ++i) l.s += t[i];
}

// the block's result, in every thread of its first warp
template <int THREADS>
__device__ __forceinline__ Lse block_join(Lse l, float (*slot)[2]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l.join(__shfl_xor_sync(0xffffffffu, l.m, o), __shfl_xor_sync(0xffffffffu, l.s, o));
    if ((threadIdx.x & 31) == 0) {
        slot[threadIdx.x >> 5][0] = l.m;
        slot[threadIdx.x >> 5][1] = l.s;
    }
    __syncthreads();
    Lse all;
    if (threadIdx.x < 32) {
        if (threadIdx.x < THREADS / 32) {
            all.m = slot[threadIdx.x][0];
            all.s = slot[threadIdx.x][1];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all.join(__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o));
    }
    return all;
}

// sums of a cluster's blocks joined in a fixed order, and x[y]; the same numbers in every lane of the calling warp and in every block. Lane = block, so that the
// loads from the others' shared memory are on their way together.
struct RowSum {
    Lse rest;      // everything but the token
    float token;   // its logit
};
__device__ __forceinline__ RowSum cluster_join(const float* mine, uint32_t blocks) {
    const uint32_t lane = threadIdx.x & 31;
    RowSum r;
    r.token = 0.f;
    float has = 0.f;
    if (lane < blocks) {
        if (blocks > 1) {
            const uint32_t peer = map_shared_rank(smem_u32(mine), lane);
            r.rest.m = ld_shared_cluster_f32(peer);
            r.rest.s = ld_shared_cluster_f32(peer + 4);
            r.token = ld_shared_cluster_f32(peer + 8);
            has = ld_shared_cluster_f32(peer + 12);
        } else {
            r.rest.m = mine[0];
            r.rest.s = mine[1];
            r.token = mine[2];
            has = mine[3];
        }
    }
    const unsigned owner = __ballot_sync(0xffffffffu, has != 0.f);
    r.token = owner ? __shfl_sync(0xffffffffu, r.token, __ffs(owner) - 1) : -INFINITY;
#pragma unroll
    for (int o = kMaxBlocks / 2; o > 0; o >>= 1) r.rest.join(__shfl_xor_sync(0xffffffffu, r.rest.m, o), __shfl_xor_sync(0xffffffffu, r.rest.s, o));
    r.rest.m = __shfl_sync(0xffffffffu, r.rest.m, 0);
    r.rest.s = __shfl_sync(0xffffffffu, r.rest.s, 0);
    return r;
}
// log of S / exp(x[y]); -inf where nothing but the token weighs. In logarithms, since a masked token's logit may be the type's lowest value
__device__ __forceinline__ double log_odds_against(const RowSum& r) { return log((double)r.rest.s) + ((double)r.rest.m - (double)r.token); }
// -log(1 + odds)
__device__ __forceinline__ double token_logprob(double log_odds) { return log_odds > 700.0 ? -log_odds : -log1p(exp(log_odds)); }

template <typename T, int THREADS, bool WIDE>
__global__ void __launch_bounds__(THREADS, 2048 / THREADS) k_token_logprobs(const T* __restrict__ logits, int64_t stride, int vocab, uint32_t blocks, int slice,
                                                             const int32_t* __restrict__ targets, float* __restrict__ logprob) {
    using P = Pack<T>;
    __shared__ float slot[THREADS / 32][2], mine[4];
    const uint32_t rank = blockIdx.x % blocks;
    const int64_t row = blockIdx.x / blocks;
    const T* src = logits + row * stride;
    const int y = targets[row], begin = min((int)rank * slice, vocab), end = min(begin + slice, vocab);
    Lse l;
    int at = begin;
    if constexpr (WIDE) {
        constexpr int U = 4;
        const int packs = (end - begin) / P::N;
        const uint4* v = (const uint4*)(src + begin);
        int i = threadIdx.x;
        for (; i + (U - 1) * THREADS < packs; i += U * THREADS) {
            uint4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = __ldcs(v + i + u * THREADS);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[P::N];
                P::unpack(raw[u], f);
                take(l, f, begin + (i + u * THREADS) * P::N, y);
            }
        }
        for (; i < packs; i += THREADS) {
            float f[P::N];
            P::unpack(__ldcs(v + i), f);
            take(l, f, begin + i * P::N, y);
        }
        at = begin + packs * P::N;
    }
    for (int i = at + threadIdx.x; i < end; i += THREADS) {
        const float f[1] = {load_one(src + i)};
        take(l, f, i, y);
    }
    const Lse all = block_join<THREADS>(l, slot);
    if (threadIdx.x == 0) {
        const bool has = y >= begin && y < end;
        mine[0] = all.m;
        mine[1] = all.s;
        mine[2] = has ? load_one(src + y) : 0.f;
        mine[3] = has ? 1.f : 0.f;
    }
    if (blocks > 1)
        cluster_sync_all();
    else
        __syncwarp();
    if (rank == 0 && threadIdx.x < 32) {
        const RowSum r = cluster_join(mine, blocks);
        if (threadIdx.x == 0) logprob[row] = (unsigned)y < (unsigned)vocab ? (float)token_logprob(log_odds_against(r)) : 0.f;
    }
    if (blocks > 1) cluster_sync_all();  // the others' results have been read
}

struct PolicyDev {
    const void* logits;
    void* d_logits;
    int64_t rows, stride;
    int vocab, slice;  // elements of a block's slice
    uint32_t blocks;   // of a cluster: of a row
    const int32_t* targets;
    const float *old_logprob, *ref_logprob, *advantage, *weight;
    float clip_low, clip_high, kl_coef;
    float *row_loss, *logprob, *kl;
    int* status;
};

// WIDE: rows start on 16 bytes. One cluster per row.
template <typename T, int THREADS, bool WIDE>
__global__ void __launch_bounds__(THREADS, THREADS > 128 ? kPerSm : 1) k_policy_loss(const __grid_constant__ PolicyDev p) {
    using P = Pack<T>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* const landed = (uint64_t*)smem;  // one barrier a piece
    float* const mine = (float*)(smem + 8 * kMaxPieces);
    T* const x_s = (T*)(smem + kHead);
    __shared__ float slot[THREADS / 32][2], coef[4];
    static_assert(8 * kMaxPieces + 16 <= kHead, "");
    pdl_launch_dependents();
    const uint32_t blocks = p.blocks, rank = blockIdx.x % blocks;
    const int64_t row = blockIdx.x / blocks;
    const T* src = (const T*)p.logits + row * p.stride;
    T* dst = p.d_logits ? (T*)p.d_logits + row * p.stride : nullptr;
    const int y = p.targets[row], begin = min((int)rank * p.slice, p.vocab), n = min(p.slice, p.vocab - begin);
    const float weight = p.weight ? p.weight[row] : 1.f;
    const int packs = WIDE ? n / P::N : 0, tid = threadIdx.x;
    if (weight == 0.f || (unsigned)y >= (unsigned)p.vocab) {  // the same in every block of the cluster
        if (rank == 0 && tid == 0) {
            if (p.logprob) p.logprob[row] = 0.f;
            if (p.row_loss) p.row_loss[row] = 0.f;
            if (p.kl) p.kl[row] = 0.f;
        }
        if (dst) {
            for (int i = tid; i < packs; i += THREADS) __stcs((uint4*)(dst + begin) + i, make_uint4(0u, 0u, 0u, 0u));
            for (int i = packs * P::N + tid; i < n; i += THREADS) store_one(dst + begin + i, 0.f);
        }
        return;
    }
    Lse l;
    if constexpr (WIDE) {
        const int bytes = packs * 16, pieces = (bytes + kPiece - 1) / kPiece;
        if (tid == 0) {
            for (int i = 0; i < pieces; ++i) mbar_init(&landed[i], 1);
            fence_mbar_init();
            for (int i = 0; i < pieces; ++i) {
                const uint32_t size = (uint32_t)min(kPiece, bytes - i * kPiece);
                mbar_arrive_expect_tx(&landed[i], size);
                bulk_g2s((uint8_t*)x_s + i * kPiece, (const uint8_t*)(src + begin) + (size_t)i * kPiece, size, &landed[i]);
            }
        }
        for (int i = packs * P::N + tid; i < n; i += THREADS) {  // less than 16 bytes at the end of the row
            const float f[1] = {load_one(src + begin + i)};
            x_s[i] = src[begin + i];
            take(l, f, begin + i, y);
        }
        __syncthreads();
        bool ok = true;
        for (int i = 0; i < pieces && ok; ++i) {
            ok = wait_barrier(&landed[i], 0, p.status, DEV_ERR_FULL_WAIT);
            const int to = min((i + 1) * (kPiece / 16), packs);
            for (int v = i * (kPiece / 16) + tid; v < to; v += THREADS) {
                float f[P::N];
                P::unpack(((const uint4*)x_s)[v], f);
                take(l, f, begin + v * P::N, y);
            }
        }
        if (!ok) let_land();
    } else {
        for (int i = tid; i < n; i += THREADS) {
            x_s[i] = src[begin + i];
            const float f[1] = {load_one(x_s + i)};
            take(l, f, begin + i, y);
        }
        __syncthreads();
    }
    const Lse all = block_join<THREADS>(l, slot);
    if (tid == 0) {
        const bool has = y >= begin && y < begin + n;
        mine[0] = all.m;
        mine[1] = all.s;
        mine[2] = has ? load_one(x_s + (y - begin)) : 0.f;
        mine[3] = has ? 1.f : 0.f;
    }
    if (blocks > 1)
        cluster_sync_all();
    else
        __syncwarp();
    if (tid < 32) {
        const RowSum r = cluster_join(mine, blocks);
        const double log_odds = log_odds_against(r), lp = token_logprob(log_odds);
        const double adv = p.advantage[row], ratio = exp(lp - (double)p.old_logprob[row]), away = p.ref_logprob ? (double)p.ref_logprob[row] - lp : 0.0;
        const double clipped = fmin(fmax(ratio, 1.0 - (double)p.clip_low), 1.0 + (double)p.clip_high) * adv;
        const double kl = away == INFINITY ? away : expm1(away) - away, free = ratio * adv;
        // a divergence of weight zero may be infinite (a masked token), and counts nothing all the same
        const double kl_loss = p.kl_coef == 0.f ? 0.0 : (double)p.kl_coef * kl, kl_slope = p.kl_coef == 0.f ? 0.0 : (double)p.kl_coef * -expm1(away);
        const double slope = (double)weight * (kl_slope - (free <= clipped ? free : 0.0));
        // p[j] = exp(x[j] - top) * share, top the row's maximum
        const float top = fmaxf(r.rest.m, r.token);
        const double share = 1.0 / ((double)r.rest.s * exp((double)r.rest.m - (double)top) + exp((double)r.token - (double)top));
        if (tid == 0) {
            coef[0] = top;
            coef[1] = (float)(-slope * share);
            coef[2] = (float)(slope / (1.0 + exp(-log_odds)));  // of the token: 1 - p[y]
        }
        if (rank == 0 && tid == 0) {
            if (p.logprob) p.logprob[row] = (float)lp;
            if (p.row_loss) p.row_loss[row] = (float)((double)weight * (kl_loss - fmin(free, clipped)));
            if (p.kl) p.kl[row] = (float)kl;
        }
    }
    __syncthreads();
    if (blocks > 1) cluster_arrive();  // this block has read the others' results
    if (dst) {
        const float top = coef[0], c = coef[1], own = coef[2];
        for (int v = tid; v < packs; v += THREADS) {
            float f[P::N];
            P::unpack(((const uint4*)x_s)[v], f);
            const int first = begin + v * P::N;
            weights(f, top);
#pragma unroll
            for (int i = 0; i < P::N; ++i) f[i] *= c;
            if ((unsigned)(y - first) < (unsigned)P::N)
#pragma unroll
                for (int i = 0; i < P::N; ++i)
                    if (first + i == y) f[i] = own;
            __stcs((uint4*)(dst + begin) + v, P::pack(f));
        }
        for (int i = packs * P::N + tid; i < n; i += THREADS)
            store_one(dst + begin + i, begin + i == y ? own : c * exp2_fast((load_one(x_s + i) - top) * kLog2e));
    }
    if (blocks > 1) cluster_wait();  // every block has read this one's result
}

// the rows' sum: fixed shares per thread, added in a fixed order, in 64 bits
__global__ void __launch_bounds__(1024) k_loss_sum(const float* row_loss, int64_t rows, float* loss) {
    __shared__ double s[32];
    pdl_wait();
    double a = 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) a += (double)row_loss[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = a;
    __syncthreads();
    if (threadIdx.x < 32) {
        a = s[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (threadIdx.x == 0) *loss = (float)a;
    }
}

// elements of a block's slice: an equal share, in whole 16-byte packs
int64_t slice_of(int64_t vocab, int blocks, int per_pack) { return ((vocab + blocks - 1) / blocks + per_pack - 1) / per_pack * per_pack; }

// Blocks of a row. Three slices fit an SM where the row allows it; with fewer rows than SMs a row is cut further, to pieces of 8 KB, so that
// more SMs fetch it.
int blocks_of(int64_t bytes, int64_t rows, int num_sms, int64_t hold) {
    int64_t n = (bytes + hold - 1) / hold;
    if (n > kMaxBlocks) n = kMaxBlocks;
    while (n < kMaxBlocks && rows * (n + 1) <= num_sms && bytes / (n + 1) >= 8192) ++n;
    return (int)std::max<int64_t>(n, 1);
}

template <typename T, int THREADS, bool WIDE>
int run_logprobs(const LossCall& c, int blocks, cudaStream_t s) {
    return (int)launch_k_cluster(k_token_logprobs<T, THREADS, WIDE>, dim3((unsigned)(c.rows * blocks)), dim3(THREADS), dim3(blocks), 0, s, false, (const T*)c.logits, c.stride,
                                 c.vocab, (uint32_t)blocks, (int)slice_of(c.vocab, blocks, Pack<T>::N), c.targets, c.logprob);
}
template <typename T>
int pick_logprobs(const LossCall& c, int num_sms, cudaStream_t s) {
    const int64_t bytes = (int64_t)c.vocab * sizeof(T);
    // a block streams a row of any length; many rows need no cluster
    const int blocks = blocks_of(bytes, c.rows, 2 * num_sms, INT64_MAX / 2);
    const bool wide = (uintptr_t)c.logits % 16 == 0 && c.stride * sizeof(T) % 16 == 0, small = bytes / blocks <= 24 * 1024;
    if (wide) return small ? run_logprobs<T, 128, true>(c, blocks, s) : run_logprobs<T, 512, true>(c, blocks, s);
    return small ? run_logprobs<T, 128, false>(c, blocks, s) : run_logprobs<T, 512, false>(c, blocks, s);
}

template <typename T, int THREADS, bool WIDE>
int run_policy(const LossCall& c, int blocks, cudaStream_t s) {
    PolicyDev p;
    p.logits = c.logits;
    p.d_logits = c.d_logits;
    p.rows = c.rows;
    p.stride = c.stride;
    p.vocab = c.vocab;
    p.slice = (int)slice_of(c.vocab, blocks, Pack<T>::N);
    p.blocks = (uint32_t)blocks;
    p.targets = c.targets;
    p.old_logprob = c.old_logprob;
    p.ref_logprob = c.ref_logprob;
    p.advantage = c.advantage;
    p.weight = c.weight;
    p.clip_low = c.clip_low;
    p.clip_high = c.clip_high;
    p.kl_coef = c.kl_coef;
    p.row_loss = c.row_loss;
    p.logprob = c.logprob;
    p.kl = c.kl;
    p.status = c.status;
    const cudaError_t e = allow_shared<k_policy_loss<T, THREADS, WIDE>>(kHead + kMaxSlice);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_k_cluster(k_policy_loss<T, THREADS, WIDE>, dim3((unsigned)(c.rows * blocks)), dim3(THREADS), dim3(blocks), kHead + (size_t)p.slice * sizeof(T), s, false, p);
}
template <typename T>
int pick_policy(const LossCall& c, int num_sms, cudaStream_t s) {
    const int64_t bytes = (int64_t)c.vocab * sizeof(T);
    const int blocks = blocks_of(bytes, c.rows, num_sms, kSharedSlice);
    const bool wide = ((uintptr_t)c.logits | (uintptr_t)c.d_logits) % 16 == 0 && c.stride * sizeof(T) % 16 == 0, small = bytes / blocks <= 24 * 1024;
    if (wide) return small ? run_policy<T, 128, true>(c, blocks, s) : run_policy<T, 256, true>(c, blocks, s);
    return small ? run_policy<T, 128, false>(c, blocks, s) : run_policy<T, 256, false>(c, blocks, s);
}

}  // namespace

bool policy_loss_supported(bool f32, int vocab) { return slice_of(vocab, kMaxBlocks, f32 ? 4 : 8) * (f32 ? 4 : 2) <= kMaxSlice; }

int launch_token_logprobs(const LossCall& c, int num_sms, cudaStream_t s) {
    if (c.rows == 0) return 0;
    return c.f32 ? pick_logprobs<float>(c, num_sms, s) : pick_logprobs<bf16>(c, num_sms, s);
}

int launch_policy_loss(const LossCall& c, int num_sms, cudaStream_t s) {
    if (c.rows == 0) return c.loss ? (int)cudaMemsetAsync(c.loss, 0, 4, s) : 0;
    const int rc = c.f32 ? pick_policy<float>(c, num_sms, s) : pick_policy<bf16>(c, num_sms, s);
    if (rc != 0 || !c.loss) return rc;
    return (int)launch_k(k_loss_sum, dim3(1), dim3(1024), 0, s, true, (const float*)c.row_loss, c.rows, c.loss);
}

}  // namespace tffn
