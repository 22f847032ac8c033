// RMS and layer norm of training rows, forward and backward. With n = (x - mean) * rstd (mean = 0 for RMS) and g = dy * weight:
//   y       = n * weight + bias
//   dx      = rstd * (g - n * mean(g * n) - mean(g)) + skip        (the last mean for the layer norm only)
//   dweight = sum over rows of dy * n,   dbias = sum over rows of dy
// A row stays in the registers of its threads, so x (and dy) are read once; statistics and sums are fp32, the variance is taken
// about the mean (two passes over registers), and a value is rounded once, when it is stored.
//
// Both are bound by HBM. Forward: a warp holds a row of up to 128 16-byte chunks, 128 threads one of up to 1 024, 512 threads a wider one;
// 8 192 x 2 048 bf16 take 14.3 us (4.7 TB/s; a row a warp 16.3 us). Backward: a persistent block walks over rows with the weight
// and its own columns of dweight / dbias in registers, the next rows on their way into shared memory; its sums go to the workspace once
// and a second kernel adds the blocks' sums per column in block order, so that the result does not depend on timing. 16 384 x 3 584 bf16
// with skip take 75 us (6.3 TB/s; loads straight into registers 97 us), 4 099 x 1 111 fp32 of the layer norm 22 us (by single
// elements 29 us).
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

// How rows lie in memory. kAligned: every row of every tensor starts on 16 bytes. kShifted: the tensors do, their rows do not; chunk c of a
// row is the c-th 16-byte unit that the row touches, so it starts `lead` columns early, and the units at the row's ends are read and
// written by element. kSingle: chunks of one element.
enum Layout { kAligned, kShifted, kSingle };

template <Layout L, int V>
__device__ __forceinline__ bool whole(int col, int width) { return L != kShifted || (col >= 0 && col + V <= width); }

// the chunk of a row from column `col` on; columns outside of the row read as 0
template <Layout L, typename T, int V>
__device__ __forceinline__ Chunk<T, V> load_chunk(const T* row, int col, int width) {
    if (whole<L, V>(col, width)) return *(const Chunk<T, V>*)(row + col);
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = (unsigned)(col + k) < (unsigned)width ? (float)row[col + k] : 0.f;
    Chunk<T, V> c;
    c.set(f);
    return c;
}
// of weight or bias, which do not shift with the rows
template <Layout L, typename T, int V>
__device__ __forceinline__ Chunk<T, V> load_weight(const T* w, int col, int width) {
    if (L != kShifted) return *(const Chunk<T, V>*)(w + col);
    float f[V];
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = (unsigned)(col + k) < (unsigned)width ? (float)w[col + k] : 0.f;
    Chunk<T, V> c;
    c.set(f);
    return c;
}
template <Layout L, typename T, int V>
__device__ __forceinline__ void store_chunk(T* row, int col, int width, const float (&f)[V]) {
    if (whole<L, V>(col, width)) {
        Chunk<T, V> c;
        c.set(f);
        *(Chunk<T, V>*)(row + col) = c;
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if ((unsigned)(col + k) < (unsigned)width) row[col + k] = (T)f[k];
    }
}

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

template <typename T, int V, bool LAYER, int TPR, int N, Layout L>
__global__ void __launch_bounds__(block_of<TPR>()) k_norm_fwd(const T* x, const T* __restrict__ w, const T* __restrict__ b, int64_t rows, int width, float eps,
                                                               T* y, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
    using C = Chunk<T, V>;
    __shared__ float slots[2][32];
    const int lane = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (block_of<TPR>() / TPR) + threadIdx.x / TPR;
    const bool live = row < rows;  // with TPR = 32 whole warps, else whole blocks
    if (TPR > 32 && !live) return;
    const T* src = x + (live ? row : 0) * width;
    const int lead = L == kShifted ? (int)((row * width) % V) : 0, end = live ? width : -V;
    auto col = [&](int i) { return (lane + i * TPR) * V - lead; };
    C v[N];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (col(i) < end) v[i] = load_chunk<L, T, V>(src, col(i), width);
    float mean = 0.f;
    if constexpr (LAYER) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col(i) < end)
#pragma unroll
                for (int k = 0; k < V; ++k) sum += v[i].get(k);
        mean = row_sum<TPR>(sum, slots[0]) / (float)width;
    }
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (col(i) < end)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = v[i].get(k) - mean;
                if (!LAYER || whole<L, V>(col(i), width) || (unsigned)(col(i) + k) < (unsigned)width) sq = fmaf(d, d, sq);
            }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, slots[1]) / (float)width + eps);
    if (!live) return;
    if (lane == 0) {
        if (LAYER && mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (col(i) >= width) break;
        const C wc = load_weight<L, T, V>(w, col(i), width);
        float out[V];
        if constexpr (LAYER) {
            const C bc = load_weight<L, T, V>(b, col(i), width);
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = fmaf((v[i].get(k) - mean) * rstd, wc.get(k), bc.get(k));
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = v[i].get(k) * rstd * wc.get(k);
        }
        store_chunk<L, T, V>(y + row * width, col(i), width, out);
    }
}

// Rows of a block are `grid` apart, and in kShifted the grid is a multiple of V (or each block has one row): `lead`, and with it the columns
// of a thread, is the same for all of them. Rows of more than a warp come through a ring of rows in shared memory, filled by
// bulk copies ahead of use; without it a block has one row's loads in flight and waits for them.
template <int V, bool LAYER, int TPR, int N, Layout L>
struct Bwd {
    static constexpr bool kRing = L != kSingle && TPR > 32 && N * TPR * 16 * 6 <= 208 * 1024;  // two rows of three tensors fit
    // resident blocks, all of them in one wave; three where four would spill the sums and the row
    static constexpr int kPerSm = TPR > 128 ? 1 : N * V * (LAYER ? 2 : 1) + (kRing ? 0 : N * V / 2) > 40 ? 3 : 4;
    static constexpr int kRows = kRing ? std::min(4, 208 * 1024 / (kPerSm * 3 * N * TPR * 16)) : 0;
};

template <typename T, int V, bool LAYER, int TPR, int N, Layout L>
__global__ void __launch_bounds__(block_of<TPR>(), Bwd<V, LAYER, TPR, N, L>::kPerSm) k_norm_bwd(const T* dy, const T* x, const T* __restrict__ w, const float* __restrict__ mean_in,
                                                               const float* __restrict__ rstd_in, const T* skip, int64_t rows, int width, T* dx,
                                                               float* __restrict__ part_w, float* __restrict__ part_b, int* status) {
    using C = Chunk<T, V>;
    constexpr int RPB = block_of<TPR>() / TPR;
    constexpr int RING = Bwd<V, LAYER, TPR, N, L>::kRows;
    __shared__ float slots[2][2][32];
    __shared__ uint64_t full[RING > 0 ? RING : 1];
    extern __shared__ __align__(128) uint8_t dynamic[];
    float* const fold = (float*)dynamic;  // RPB > 1: [RPB][width] sums of the warps
    const int pitch = L == kShifted ? (width + 2 * V - 2) / V * V : width;
    T* const ring = (T*)dynamic;  // [RING][dy, x, skip][pitch], a row from the 16-byte unit on in which it begins
    pdl_launch_dependents();
    const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t first = (int64_t)blockIdx.x * RPB + sub, step = (int64_t)gridDim.x * RPB;
    const int lead = L == kShifted ? (int)((first * width) % V) : 0;
    const float inv = 1.f / (float)width;
    auto col = [&](int i) { return (lane + i * TPR) * V - lead; };
    auto fetch = [&](int64_t row, int stage) {  // by one thread
        T* const to = ring + (size_t)stage * 3 * pitch;
        int units = (lead + width + V - 1) / V;
        // the unit in which the last row ends may reach behind the tensors
        if (L == kShifted && row + 1 == rows) {
            units = (lead + width) / V;
            for (int c = units * V; c < lead + width; ++c) {
                to[c] = dy[row * width - lead + c];
                to[pitch + c] = x[row * width - lead + c];
                if (skip) to[2 * pitch + c] = skip[row * width - lead + c];
            }
        }
        const uint32_t bytes = (uint32_t)units * 16;
        mbar_arrive_expect_tx(&full[stage], skip ? 3 * bytes : 2 * bytes);
        if (units == 0) return;
        bulk_g2s(to, dy + row * width - lead, bytes, &full[stage]);
        bulk_g2s(to + pitch, x + row * width - lead, bytes, &full[stage]);
        if (skip) bulk_g2s(to + 2 * pitch, skip + row * width - lead, bytes, &full[stage]);
    };
    if (RING && threadIdx.x == 0) {
        for (int i = 0; i < RING; ++i) mbar_init(&full[i], 1);
        fence_mbar_init();
        for (int i = 0; i < RING; ++i)
            if (first + i * step < rows) fetch(first + i * step, i);
    }
    C wv[N];
    float aw[N][V], ab[LAYER ? N : 1][V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (col(i) < width) wv[i] = load_weight<L, T, V>(w, col(i), width);
#pragma unroll
        for (int k = 0; k < V; ++k) aw[i][k] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < (LAYER ? N : 1); ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) ab[i][k] = 0.f;
    int turn = 0, stage = 0, phase = 0;
    bool ok = true;
    float rstd_next = first < rows ? rstd_in[first] : 0.f, mean_next = LAYER && first < rows ? mean_in[first] : 0.f;
    if (RING) __syncthreads();
    for (int64_t row = first; row < rows; row += step, turn ^= 1) {
        C dv[N], xv[N], sv[N];
        const float rstd = rstd_next, mean = mean_next;
        if (row + step < rows) {
            rstd_next = rstd_in[row + step];
            if (LAYER) mean_next = mean_in[row + step];
        }
        if (RING) ok = ok && wait_barrier(&full[stage], phase, status, DEV_ERR_FULL_WAIT);
        const T* const src_d = RING ? ring + (size_t)stage * 3 * pitch + lead : dy + row * width;
        const T* const src_x = RING ? src_d + pitch : x + row * width;
        const T* const src_s = RING ? src_d + 2 * pitch : skip + row * width;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col(i) < width) {
                dv[i] = load_chunk<L, T, V>(src_d, col(i), width);
                xv[i] = load_chunk<L, T, V>(src_x, col(i), width);
            }
        if (skip)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (col(i) < width) sv[i] = load_chunk<L, T, V>(src_s, col(i), width);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (col(i) < width)
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
            if (RING && threadIdx.x == 0 && ok && row + RING * step < rows) fetch(row + RING * step, stage);  // every thread has its part of the row
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
            if (col(i) < width) {
                float out[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float n = (xv[i].get(k) - mean) * rstd, g = dv[i].get(k) * wv[i].get(k);
                    out[k] = rstd * (LAYER ? fmaf(-n, s1, g) - s2 : fmaf(-n, s1, g));
                    if (skip) out[k] += sv[i].get(k);
                }
                store_chunk<L, T, V>(dx + row * width, col(i), width, out);
            }
        if (RING && ++stage == RING) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (RING && !ok) let_land();
    if (!part_w && !part_b) return;
    // with kShifted rows each warp has columns of its own, so its sums are added by column in shared memory
    auto leave = [&](float(&a)[N][V], float* part) {
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if ((unsigned)(col(i) + k) < (unsigned)width) fold[(size_t)sub * width + col(i) + k] = a[i][k];
            __syncthreads();
            for (int c = threadIdx.x; c < width; c += block_of<TPR>()) {
                float t = 0.f;
#pragma unroll
                for (int r = 0; r < RPB; ++r) t += fold[(size_t)r * width + c];
                part[(size_t)blockIdx.x * width + c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if constexpr (L == kAligned) {
                    if (col(i) < width)
#pragma unroll
                        for (int k = 0; k < V; k += 4)
                            *(float4*)(part + (size_t)blockIdx.x * width + col(i) + k) = make_float4(a[i][k], a[i][k + 1], a[i][k + 2], a[i][k + 3]);
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k)
                        if ((unsigned)(col(i) + k) < (unsigned)width) part[(size_t)blockIdx.x * width + col(i) + k] = a[i][k];
                }
        }
    };
    if (part_w) leave(aw, part_w);
    if constexpr (LAYER)
        if (part_b) leave(ab, part_b);
}

// column sums of the blocks' parts, in block order: kRuns runs of blocks per column, added in order
constexpr int kRuns = 32;
static_assert(kMaxParts % kRuns == 0, "");
__global__ void __launch_bounds__(32 * kRuns) k_norm_fold(const float* part_w, const float* part_b, int parts, int width, float* dweight, float* dbias) {
    __shared__ float s[kRuns][33];
    pdl_wait();
    const float* part = blockIdx.y ? part_b : part_w;
    float* out = blockIdx.y ? dbias : dweight;
    const int col = blockIdx.x * 32 + threadIdx.x, run = (parts + kRuns - 1) / kRuns, p0 = threadIdx.y * run, p1 = min(p0 + run, parts);
    float a = 0.f;
    if (col < width) {
        float v[kMaxParts / kRuns];  // all of them in flight
#pragma unroll
        for (int i = 0; i < kMaxParts / kRuns; ++i) v[i] = p0 + i < p1 ? part[(size_t)(p0 + i) * width + col] : 0.f;
#pragma unroll
        for (int i = 0; i < kMaxParts / kRuns; ++i) a += v[i];
    }
    s[threadIdx.y][threadIdx.x] = a;
    __syncthreads();
    if (threadIdx.y == 0 && col < width) {
        a = 0.f;
#pragma unroll
        for (int i = 0; i < kRuns; ++i) a += s[i][threadIdx.x];
        out[col] = a;
    }
}

// 16-byte chunks that a row of the width can touch
template <int V, Layout L>
int chunks_of(int width) { return L == kShifted ? (width + 2 * V - 2) / V : width / V; }

template <typename T, int V, bool LAYER, int TPR, int N, Layout L>
int run_fwd(const NormCall& c, cudaStream_t s) {
    constexpr int RPB = block_of<TPR>() / TPR;
    const int64_t blocks = (c.rows + RPB - 1) / RPB;
    return (int)launch_k(k_norm_fwd<T, V, LAYER, TPR, N, L>, dim3((unsigned)blocks), dim3(block_of<TPR>()), 0, s, false, (const T*)c.x, (const T*)c.weight, (const T*)c.bias,
                         c.rows, c.width, c.eps, (T*)c.y, c.mean, c.rstd);
}

template <typename T, int V, bool LAYER, int TPR, int N, Layout L>
int run_bwd(const NormCall& c, int num_sms, cudaStream_t s) {
    constexpr int RPB = block_of<TPR>() / TPR;
    using B = Bwd<V, LAYER, TPR, N, L>;
    constexpr int RING = B::kRows;
    const size_t shared = RING ? (size_t)3 * RING * chunks_of<V, L>(c.width) * 16 : RPB > 1 ? (size_t)RPB * c.width * 4 : 0;
    auto kernel = k_norm_bwd<T, V, LAYER, TPR, N, L>;
    if (RING) {
        const cudaError_t e = allow_shared<k_norm_bwd<T, V, LAYER, TPR, N, L>>(3 * RING * N * TPR * 16);
        if (e != cudaSuccess) return (int)e;
    }
    int parts = (int)std::min<int64_t>((c.rows + RPB - 1) / RPB, std::min(kMaxParts, num_sms * B::kPerSm));
    if (L == kShifted && c.rows > (int64_t)parts * RPB) parts = (int)std::max<int64_t>(parts / V * V, std::min<int64_t>(V, (c.rows + RPB - 1) / RPB));
    const bool fold = c.dweight || c.dbias;
    float* part_w = c.dweight ? c.workspace : nullptr;
    float* part_b = c.dbias ? c.workspace + (size_t)parts * c.width : nullptr;
    int rc = (int)launch_k(kernel, dim3(parts), dim3(block_of<TPR>()), shared, s, false, (const T*)c.dy, (const T*)c.x, (const T*)c.weight, (const float*)c.mean,
                           (const float*)c.rstd, (const T*)c.skip, c.rows, c.width, (T*)c.dx, part_w, part_b, c.status);
    if (rc == 0 && fold) {
        // blockIdx.y: dweight, dbias; a missing one is skipped by its own launch shape
        if (c.dweight && c.dbias)
            rc = (int)launch_k(k_norm_fold, dim3((c.width + 31) / 32, 2), dim3(32, kRuns), 0, s, true, (const float*)part_w, (const float*)part_b, parts, c.width, c.dweight, c.dbias);
        else
            rc = (int)launch_k(k_norm_fold, dim3((c.width + 31) / 32, 1), dim3(32, kRuns), 0, s, true, (const float*)(c.dweight ? part_w : part_b), (const float*)nullptr, parts,
                               c.width, c.dweight ? c.dweight : c.dbias, (float*)nullptr);
    }
    return rc;
}

template <typename T, int V, bool LAYER, Layout L>
int pick_fwd(const NormCall& c, cudaStream_t s) {
    const int chunks = chunks_of<V, L>(c.width);
    if (chunks <= 64) return run_fwd<T, V, LAYER, 32, 2, L>(c, s);
    if (chunks <= 128) return run_fwd<T, V, LAYER, 32, 4, L>(c, s);
    if (chunks <= 256) return run_fwd<T, V, LAYER, 128, 2, L>(c, s);
    if (chunks <= 512) return run_fwd<T, V, LAYER, 128, 4, L>(c, s);
    if (chunks <= 1024) return run_fwd<T, V, LAYER, 128, 8, L>(c, s);
    if (chunks <= 2048) return run_fwd<T, V, LAYER, 512, 4, L>(c, s);
    if constexpr (V < 8)  // kNormMaxWidth is 2 048 chunks of 8
        if (chunks <= 4096) return run_fwd<T, V, LAYER, 512, 8, L>(c, s);
    if constexpr (V == 1) return run_fwd<T, V, LAYER, 512, 32, L>(c, s);
    return (int)cudaErrorInvalidValue;
}

template <typename T, int V, bool LAYER, Layout L>
int pick_bwd(const NormCall& c, int num_sms, cudaStream_t s) {
    const int chunks = chunks_of<V, L>(c.width);
    if (chunks <= 64) return run_bwd<T, V, LAYER, 32, 2, L>(c, num_sms, s);
    if (chunks <= 128) return run_bwd<T, V, LAYER, 32, 4, L>(c, num_sms, s);
    if (chunks <= 256) return run_bwd<T, V, LAYER, 128, 2, L>(c, num_sms, s);
    if (chunks <= 512) return run_bwd<T, V, LAYER, 128, 4, L>(c, num_sms, s);
    if (chunks <= 1024) return run_bwd<T, V, LAYER, 512, 2, L>(c, num_sms, s);
    if (chunks <= 2048) return run_bwd<T, V, LAYER, 512, 4, L>(c, num_sms, s);
    if constexpr (V < 8)
        if (chunks <= 4096) return run_bwd<T, V, LAYER, 512, 8, L>(c, num_sms, s);
    if constexpr (V == 1) return run_bwd<T, V, LAYER, 512, 32, L>(c, num_sms, s);
    return (int)cudaErrorInvalidValue;
}

template <typename T, int V>
Layout layout_of(const NormCall& c) {
    const uintptr_t rows = (uintptr_t)c.x | (uintptr_t)c.y | (uintptr_t)c.dy | (uintptr_t)c.skip | (uintptr_t)c.dx;
    const uintptr_t weights = (uintptr_t)c.weight | (uintptr_t)c.bias;
    if (rows % 16 != 0) return kSingle;
    if (c.width % V == 0 && weights % 16 == 0) return kAligned;
    return chunks_of<V, kShifted>(c.width) <= kNormMaxWidth / V ? kShifted : kSingle;
}

template <typename T, int V, bool LAYER>
int forward(const NormCall& c, cudaStream_t s) {
    switch (layout_of<T, V>(c)) {
        case kAligned: return pick_fwd<T, V, LAYER, kAligned>(c, s);
        case kShifted: return pick_fwd<T, V, LAYER, kShifted>(c, s);
        default: return pick_fwd<T, 1, LAYER, kSingle>(c, s);
    }
}
template <typename T, int V, bool LAYER>
int backward(const NormCall& c, int num_sms, cudaStream_t s) {
    switch (layout_of<T, V>(c)) {
        case kAligned: return pick_bwd<T, V, LAYER, kAligned>(c, num_sms, s);
        case kShifted: return pick_bwd<T, V, LAYER, kShifted>(c, num_sms, s);
        default: return pick_bwd<T, 1, LAYER, kSingle>(c, num_sms, s);
    }
}

}  // namespace

int64_t norm_workspace_floats(int64_t rows, int width) { return 2 * std::min<int64_t>(rows, kMaxParts) * width; }

int launch_norm_forward(const NormCall& c, int, cudaStream_t s) {
    if (c.rows == 0) return 0;
    if (c.f32) return c.layer ? forward<float, 4, true>(c, s) : forward<float, 4, false>(c, s);
    return c.layer ? forward<bf16, 8, true>(c, s) : forward<bf16, 8, false>(c, s);
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
    if (c.f32) return c.layer ? backward<float, 4, true>(c, num_sms, s) : backward<float, 4, false>(c, num_sms, s);
    return c.layer ? backward<bf16, 8, true>(c, num_sms, s) : backward<bf16, 8, false>(c, num_sms, s);
}

}  // namespace tffn
