// RMS and layer norm of training rows, forward and backward. With n = (x - mean) * rstd (mean = 0 for RMS) and g = dy * weight:
//   y       = n * weight + bias
//   dx      = rstd * (g - n * mean(g * n) - mean(g)) + skip        (the last mean for the layer norm only)
//   dweight = sum over rows of dy * n,   dbias = sum over rows of dy
// A row stays in the registers of its threads, so x (and dy) are read once; statistics and sums are fp32, the variance is taken
// about the mean (two passes over registers), and a value is rounded once, when it is stored.
//
// Both are bound by HBM. Forward: a block of 128 threads holds four rows (up to 256 16-byte chunks wide), one row, or a block of 512 one
// row. Backward: a persistent block walks over rows with the weight and its own columns of dweight / dbias in registers; its sums go to
// the workspace once and a second kernel adds the blocks' sums per column in block order, so that the result does not depend on timing.
#include "launch.h"
#include "ptx.cuh"
#include "train.h"
#include <algorithm>

namespace tffn {

namespace {

constexpr int kMaxParts = 640;  // blocks of the backward pass, at most

// V consecutive elements in the memory format: 16 bytes, or one element where rows are not 16-byte aligned
template <typename T, int V>
struct Chunk;
template <>
struct Chunk<float, 4> {
    float4 v;
    __device__ __forceinline__ float get(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
    __device__ __forceinline__ void set(const float (&f)[4]) { v = make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Chunk<bf16, 8> {
    uint4 v;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return i & 1 ? bf16_hi(w) : bf16_lo(w);
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]), c = __floats2bfloat162_rn(f[4], f[5]),
                             d = __floats2bfloat162_rn(f[6], f[7]);
        v = make_uint4(*(const uint32_t*)&a, *(const uint32_t*)&b, *(const uint32_t*)&c, *(const uint32_t*)&d);
    }
};
template <>
struct Chunk<float, 1> {
    float v;
    __device__ __forceinline__ float get(int) const { return v; }
    __device__ __forceinline__ void set(const float (&f)[1]) { v = f[0]; }
};
template <>
struct Chunk<bf16, 1> {
    bf16 v;
    __device__ __forceinline__ float get(int) const { return __bfloat162float(v); }
    __device__ __forceinline__ void set(const float (&f)[1]) { v = __float2bfloat16_rn(f[0]); }
};

// sum over the TPR threads of a row; slot: 32 floats of shared memory per call site that may still be read
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* slot) {
    v = warp_sum(v);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) v += slot[i];
    }
    return v;
}

template <int TPR>
constexpr int block_of() { return TPR > 128 ? TPR : 128; }

template <typename T, int V, bool LAYER, int TPR, int N>
__global__ void __launch_bounds__(block_of<TPR>()) k_norm_fwd(const T* x, const T* __restrict__ w, const T* __restrict__ b, int64_t rows, int width, float eps,
                                                               T* y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    using C = Chunk<T, V>;
    __shared__ float slots[2][32];
    const int lane = threadIdx.x % TPR, chunks = width / V;
    const int64_t row = (int64_t)blockIdx.x * (block_of<TPR>() / TPR) + threadIdx.x / TPR;
    const bool live = row < rows;  // with TPR = 32 whole warps, else whole blocks
    if (TPR > 32 && !live) return;
    const C* src = (const C*)(x + (live ? row : 0) * width);
    C v[N];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane + i * TPR < chunks && live) v[i] = src[lane + i * TPR];
    float mean = 0.f;
    if constexpr (LAYER) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + i * TPR < chunks && live)
#pragma unroll
                for (int k = 0; k < V; ++k) sum += v[i].get(k);
        mean = row_sum<TPR>(sum, slots[0]) / (float)width;
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (lane + i * TPR < chunks && live)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = v[i].get(k) - mean;
                sq = fmaf(d, d, sq);
            }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, slots[1]) / (float)width + eps);
    if (!live) return;
    if (lane == 0) {
        if (LAYER && mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    C* dst = (C*)(y + row * width);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = lane + i * TPR;
        if (c >= chunks) break;
        const C wc = ((const C*)w)[c];
        float out[V];
        if constexpr (LAYER) {
            const C bc = ((const C*)b)[c];
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = fmaf((v[i].get(k) - mean) * rstd, wc.get(k), bc.get(k));
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = v[i].get(k) * rstd * wc.get(k);
        }
        C o;
        o.set(out);
        dst[c] = o;
    }
}

template <typename T, int V, bool LAYER, int TPR, int N>
__global__ void __launch_bounds__(block_of<TPR>()) k_norm_bwd(const T* dy, const T* x, const T* __restrict__ w, const float* __restrict__ mean_in,
                                                               const float* __restrict__ rstd_in, const T* skip, int64_t rows, int width, T* dx,
                                                               float* __restrict__ part_w, float* __restrict__ part_b) {
    using C = Chunk<T, V>;
    constexpr int RPB = block_of<TPR>() / TPR;
    __shared__ float slots[2][2][32];
    extern __shared__ float fold[];  // RPB > 1: [RPB - 1][width] sums of the other warps
    pdl_launch_dependents();
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR, chunks = width / V;
    const float inv = 1.f / (float)width;
    C wv[N];
    float aw[N][V], ab[LAYER ? N : 1][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (lane + i * TPR < chunks) wv[i] = ((const C*)w)[lane + i * TPR];
#pragma unroll
        for (int k = 0; k < V; ++k) aw[i][k] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < (LAYER ? N : 1); ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) ab[i][k] = 0.f;
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < rows; row += (int64_t)gridDim.x * RPB, turn ^= 1) {
        C dv[N], xv[N], sv[N];
        const float rstd = rstd_in[row], mean = LAYER ? mean_in[row] : 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + i * TPR < chunks) {
                dv[i] = ((const C*)(dy + row * width))[lane + i * TPR];
                xv[i] = ((const C*)(x + row * width))[lane + i * TPR];
            }
        if (skip)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + i * TPR < chunks) sv[i] = ((const C*)(skip + row * width))[lane + i * TPR];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + i * TPR < chunks)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = dv[i].get(k), n = (xv[i].get(k) - mean) * rstd, g = d * wv[i].get(k);
                    s1 = fmaf(g, n, s1);
                    aw[i][k] = fmaf(d, n, aw[i][k]);
                    if constexpr (LAYER) {
                        s2 += g;
                        ab[i][k] += d;
                    }
                }
        // a slot is written again two rows later, behind the barrier of the row between
        if constexpr (TPR > 32) {
            s1 = warp_sum(s1);
            if constexpr (LAYER) s2 = warp_sum(s2);
            if ((threadIdx.x & 31) == 0) {
                slots[turn][0][threadIdx.x >> 5] = s1;
                if constexpr (LAYER) slots[turn][1][threadIdx.x >> 5] = s2;
            }
            __syncthreads();
            s1 = s2 = 0.f;
#pragma unroll
            for (int i = 0; i < TPR / 32; ++i) {
                s1 += slots[turn][0][i];
                if constexpr (LAYER) s2 += slots[turn][1][i];
            }
        } else {
            s1 = warp_sum(s1);
            if constexpr (LAYER) s2 = warp_sum(s2);
        }
        s1 *= inv;
        s2 *= inv;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + i * TPR < chunks) {
                float out[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float n = (xv[i].get(k) - mean) * rstd, g = dv[i].get(k) * wv[i].get(k);
                    out[k] = rstd * (LAYER ? fmaf(-n, s1, g) - s2 : fmaf(-n, s1, g));
                    if (skip) out[k] += sv[i].get(k);
                }
                C o;
                o.set(out);
                ((C*)(dx + row * width))[lane + i * TPR] = o;
            }
    }
    if (!part_w && !part_b) return;
    auto leave = [&](float(&a)[N][V], float* part) {
        if constexpr (RPB > 1) {
            __syncthreads();
            if (sub > 0)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (lane + i * TPR < chunks)
#pragma unroll
                        for (int k = 0; k < V; ++k) fold[(size_t)(sub - 1) * width + (lane + i * TPR) * V + k] = a[i][k];
            __syncthreads();
            if (sub > 0) return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + i * TPR < chunks)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int c = (lane + i * TPR) * V + k;
                    float t = a[i][k];
                    for (int r = 0; r < RPB - 1; ++r) t += fold[(size_t)r * width + c];
                    part[(size_t)blockIdx.x * width + c] = t;
                }
    };
    if (part_w) leave(aw, part_w);
    if constexpr (LAYER)
        if (part_b) leave(ab, part_b);
}

// column sums of the blocks' parts, in block order: 16 runs of blocks per column, added in order
__global__ void __launch_bounds__(512) k_norm_fold(const float* part_w, const float* part_b, int parts, int width, float* dweight, float* dbias) {
    __shared__ float s[16][33];
    pdl_wait();
    const float* part = blockIdx.y ? part_b : part_w;
    float* out = blockIdx.y ? dbias : dweight;
    const int col = blockIdx.x * 32 + threadIdx.x, run = (parts + 15) / 16, p0 = threadIdx.y * run, p1 = min(p0 + run, parts);
    float a = 0.f;
    if (col < width)
#pragma unroll 8
        for (int p = p0; p < p1; ++p) a += part[(size_t)p * width + col];
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && col < width) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) a += s[i][threadIdx.x];
        out[col] = a;
    }
}

template <typename T, int V, bool LAYER, int TPR, int N>
int run_fwd(const NormCall& c, cudaStream_t s) {
    constexpr int RPB = block_of<TPR>() / TPR;
    const int64_t blocks = (c.rows + RPB - 1) / RPB;
    return (int)launch_k(k_norm_fwd<T, V, LAYER, TPR, N>, dim3((unsigned)blocks), dim3(block_of<TPR>()), 0, s, false, (const T*)c.x, (const T*)c.weight, (const T*)c.bias, c.rows,
                         c.width, c.eps, (T*)c.y, c.mean, c.rstd);
}

template <typename T, int V, bool LAYER, int TPR, int N>
int run_bwd(const NormCall& c, int num_sms, cudaStream_t s) {
    constexpr int RPB = block_of<TPR>() / TPR;
    const int parts = (int)std::min<int64_t>((c.rows + RPB - 1) / RPB, std::min(kMaxParts, num_sms * (TPR > 128 ? 2 : 4)));
    const bool fold = c.dweight || c.dbias;
    float* part_w = c.dweight ? c.workspace : nullptr;
    float* part_b = c.dbias ? c.workspace + (size_t)parts * c.width : nullptr;
    int rc = (int)launch_k(k_norm_bwd<T, V, LAYER, TPR, N>, dim3(parts), dim3(block_of<TPR>()), (size_t)(RPB - 1) * c.width * 4, s, false, (const T*)c.dy, (const T*)c.x,
                           (const T*)c.weight, (const float*)c.mean, (const float*)c.rstd, (const T*)c.skip, c.rows, c.width, (T*)c.dx, part_w, part_b);
    if (rc == 0 && fold) {
        // blockIdx.y: dweight, dbias; a missing one is skipped by its own launch shape
        if (c.dweight && c.dbias)
            rc = (int)launch_k(k_norm_fold, dim3((c.width + 31) / 32, 2), dim3(32, 16), 0, s, true, (const float*)part_w, (const float*)part_b, parts, c.width, c.dweight, c.dbias);
        else
            rc = (int)launch_k(k_norm_fold, dim3((c.width + 31) / 32, 1), dim3(32, 16), 0, s, true, (const float*)(c.dweight ? part_w : part_b), (const float*)nullptr, parts,
                               c.width, c.dweight ? c.dweight : c.dbias, (float*)nullptr);
    }
    return rc;
}

template <typename T, int V, bool LAYER>
int pick_fwd(const NormCall& c, cudaStream_t s) {
    const int chunks = c.width / V;
    if (chunks <= 64) return run_fwd<T, V, LAYER, 32, 2>(c, s);
    if (chunks <= 128) return run_fwd<T, V, LAYER, 32, 4>(c, s);
    if (chunks <= 256) return run_fwd<T, V, LAYER, 32, 8>(c, s);
    if (chunks <= 512) return run_fwd<T, V, LAYER, 128, 4>(c, s);
    if (chunks <= 1024) return run_fwd<T, V, LAYER, 128, 8>(c, s);
    if (chunks <= 2048) return run_fwd<T, V, LAYER, 512, 4>(c, s);
    if constexpr (V < 8)  // kNormMaxWidth is 2 048 chunks of 8
        if (chunks <= 4096) return run_fwd<T, V, LAYER, 512, 8>(c, s);
    if constexpr (V == 1) return run_fwd<T, V, LAYER, 512, 32>(c, s);
    return (int)cudaErrorInvalidValue;
}

template <typename T, int V, bool LAYER>
int pick_bwd(const NormCall& c, int num_sms, cudaStream_t s) {
    const int chunks = c.width / V;
    if (chunks <= 64) return run_bwd<T, V, LAYER, 32, 2>(c, num_sms, s);
    if (chunks <= 128) return run_bwd<T, V, LAYER, 32, 4>(c, num_sms, s);
    if (chunks <= 256) return run_bwd<T, V, LAYER, 128, 2>(c, num_sms, s);
    if (chunks <= 512) return run_bwd<T, V, LAYER, 128, 4>(c, num_sms, s);
    if (chunks <= 1024) return run_bwd<T, V, LAYER, 512, 2>(c, num_sms, s);
    if (chunks <= 2048) return run_bwd<T, V, LAYER, 512, 4>(c, num_sms, s);
    if constexpr (V < 8)
        if (chunks <= 4096) return run_bwd<T, V, LAYER, 512, 8>(c, num_sms, s);
    if constexpr (V == 1) return run_bwd<T, V, LAYER, 512, 32>(c, num_sms, s);
    return (int)cudaErrorInvalidValue;
}

// 16-byte accesses where every row of every tensor starts on 16 bytes
bool wide_rows(const NormCall& c, int per_chunk) {
    const uintptr_t all = (uintptr_t)c.x | (uintptr_t)c.weight | (uintptr_t)c.bias | (uintptr_t)c.y | (uintptr_t)c.dy | (uintptr_t)c.skip | (uintptr_t)c.dx;
    return c.width % per_chunk == 0 && all % 16 == 0;
}

}  // namespace

int64_t norm_workspace_floats(int64_t rows, int width) { return 2 * std::min<int64_t>(rows, kMaxParts) * width; }

int launch_norm_forward(const NormCall& c, int, cudaStream_t s) {
    if (c.rows == 0) return 0;
    if (c.f32) {
        if (wide_rows(c, 4)) return c.layer ? pick_fwd<float, 4, true>(c, s) : pick_fwd<float, 4, false>(c, s);
        return c.layer ? pick_fwd<float, 1, true>(c, s) : pick_fwd<float, 1, false>(c, s);
    }
    if (wide_rows(c, 8)) return c.layer ? pick_fwd<bf16, 8, true>(c, s) : pick_fwd<bf16, 8, false>(c, s);
    return c.layer ? pick_fwd<bf16, 1, true>(c, s) : pick_fwd<bf16, 1, false>(c, s);
}

int launch_norm_backward(const NormCall& c, int num_sms, cudaStream_t s) {
    if (c.rows == 0) {  // no rows: the sums are zero
        for (float* p : {c.dweight, c.dbias})
            if (p) {
                const cudaError_t e = cudaMemsetAsync(p, 0, (size_t)c.width * 4, s);
                if (e != cudaSuccess) return (int)e;
            }
        return 0;
    }
    if (c.f32) {
        if (wide_rows(c, 4)) return c.layer ? pick_bwd<float, 4, true>(c, num_sms, s) : pick_bwd<float, 4, false>(c, num_sms, s);
        return c.layer ? pick_bwd<float, 1, true>(c, num_sms, s) : pick_bwd<float, 1, false>(c, num_sms, s);
    }
    if (wide_rows(c, 8)) return c.layer ? pick_bwd<bf16, 8, true>(c, num_sms, s) : pick_bwd<bf16, 8, false>(c, num_sms, s);
    return c.layer ? pick_bwd<bf16, 1, true>(c, num_sms, s) : pick_bwd<bf16, 1, false>(c, num_sms, s);
}

}  // namespace tffn
