// Attention of packed training sequences on the tensor cores, forward and backward. With P = exp(scale Q K^T - lse) inside the mask and 0
// outside, D = rowsum(dO o O):
//   O = P V,   lse = log rowsum exp(scale Q K^T)
//   dS = P o (dO V^T - D),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
// The backward pass forms P again from lse, so nothing of the size queries x keys is ever stored.
//
// One shape serves all three kernels. 128 rows stand still (queries for O and dQ, keys for dK and dV) while tiles of 64 rows of the other
// side stream past through a ring that one warp fills by TMA:
//   forward   S = Q K^T                       | O  += P V
//   dQ        S = Q K^T,   dP = dO V^T        | dQ += dS K
//   dK, dV    S^T = K Q^T, dP^T = V dO^T      | dV += P^T dO,  dK += dS^T Q
// The left products take both operands along the head; the right ones take the streamed tile a second time, read the other way round, and
// P or dS from the tensor memory that S or dP came from, in bf16. Standing operands lie in tensor memory, where they cost no
// shared-memory bandwidth (in shared memory for dK, dV of 128-wide heads, which leave no room there). Thread = standing row, so that a
// row's mask is one interval of columns and its statistics need no exchange. Two groups of four warps take alternate tiles; one's exponentials run
// under the other's products. In the forward pass each group has a maximum, a sum and an O of its own, joined at the end.
//
// P and dS enter their products as bf16: half a step, 2^-9 of each term, the rounding that inputs and results have as well; S, dP, sums,
// statistics and O, dQ, dK, dV are fp32 until they are stored.
//
// dQ and dK, dV are two kernels, each with its own S and dP: 7 products of a tile instead of 5, but every output row has one block that
// adds it up in one order, so the gradients are the same bits on every run, without atomics on dQ.
#include "launch.h"
#include "ptx.cuh"
#include "train.h"
#include <cmath>
#include <cstring>

namespace tffn {

namespace {

constexpr int kStand = 128, kTile = 64, kWarpsOfGroup = 4, kThreads = 320;
constexpr float kLog2e = 1.4426950408889634f;
enum Kind { FWD = 0, DQ = 1, DKV = 2 };

template <int HD, int KIND>
struct Cfg {
    static constexpr int BLOCKS = HD / 64;                   // column blocks of 64 (128 swizzled bytes)
    static constexpr int BLOCK = kTile * 128, TILE = BLOCKS * BLOCK, STAGE = 2 * TILE;
    static constexpr bool A_SHARED = KIND == DKV && HD == 128;
    static constexpr int A_BLOCK = kStand * 128, A_TILE = A_SHARED ? BLOCKS * A_BLOCK : 0;
    static constexpr int STAGES = 4;
    static constexpr int RING = 2 * A_TILE, AFTER = RING + STAGES * STAGE;
    static constexpr int BARS = AFTER, ROWS = BARS + 256;    // ROWS: lse and D of streamed queries, or the groups' statistics
    static constexpr int SMEM = ROWS + 2 * 2 * kTile * 8;
    // tensor memory columns
    static constexpr int A0 = 0, A1 = HD / 2;
    static constexpr int S = A_SHARED ? 0 : KIND == FWD ? HD / 2 : HD;
    static constexpr int S_STEP = KIND == FWD ? kTile : 2 * kTile;         // S, and dP behind it
    static constexpr int P = S + 2 * kTile;                                // forward only (32 columns a group); else P and dS lie where S and dP were
    static constexpr int ACC = KIND == FWD ? P + kTile : S + 4 * kTile;    // O of each group; dQ; dK, dV
    static constexpr int COLS = ACC + (KIND == DQ ? HD : 2 * HD);
    static_assert(COLS <= 512 && SMEM <= 227 * 1024, "");
};

struct Dev {
    CUtensorMap tm[2];   // streamed operands: K, V or Q, dO; boxes of 64 rows x 64 columns of one head
    CUtensorMap tmA[2];  // standing K, V where they lie in shared memory; boxes of 128 rows
    const bf16 *a0, *a1; // standing rows: Q, dO or K, V
    int64_t a0_stride, a1_stride;
    const int *cu_q, *cu_k;
    int64_t rows_q, rows_k;
    int max_q, max_k, n_seqs, heads, kv_heads, hd, causal, chunk;
    int parts;           // of the query heads of a kv head (dK, dV)
    float scale, scale_log2;
    float* lse;          // [heads][rows_q]
    const float* d;      // [heads][rows_q]
    bf16 *out0, *out1;   // O; dQ; dK, dV
    int64_t out0_stride, out1_stride;
    float* partial;      // parts > 1: dK, dV as fp32 [2][parts][rows_k][kv_heads][hd]
    int* status;
};

struct Span {
    int64_t first;
    int len;
};
// rows of sequence i, whatever the offsets say inside the buffer and not longer than promised
__device__ __forceinline__ Span span_of(const int* cu, int i, int64_t rows, int most) {
    const int64_t b = min(max((int64_t)cu[i], (int64_t)0), rows), e = min(max((int64_t)cu[i + 1], b), rows);
    return {b, (int)min(e - b, (int64_t)most)};
}

__device__ __forceinline__ void group_barrier(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
__device__ __forceinline__ void groups_barrier() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}

// a standing row (or zeros) into the calling lane's tensor memory, two columns of the head per word
template <int HD>
__device__ __forceinline__ void row_to_tmem(uint32_t taddr, const bf16* row, int hd) {
#pragma unroll
    for (int c = 0; c < HD; c += 32) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (row && c + 8 * i < hd) v = __ldg((const uint4*)(row + c + 8 * i));
            w[4 * i] = v.x;
            w[4 * i + 1] = v.y;
            w[4 * i + 2] = v.z;
            w[4 * i + 3] = v.w;
        }
        tmem_st16(taddr + c / 2, w);
    }
    tc_wait_st();
}

template <int HD, int KIND>
__global__ void __launch_bounds__(kThreads, 1) k_train_attn(const __grid_constant__ Dev p) {
    using C = Cfg<HD, KIND>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* const full = (uint64_t*)(smem + C::BARS);
    uint64_t *const empty = full + C::STAGES, *const s_full = empty + C::STAGES, *const s_free = s_full + 2, *const p_full = s_free + 2, *const p_done = p_full + 2,
                    *const a_full = p_done + 2, *const all_done = a_full + 1;
    uint32_t* const tmem_slot = (uint32_t*)(all_done + 1);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;

    // ---- what this block computes
    int unit = blockIdx.x;
    const int fast = KIND == DKV ? p.kv_heads * p.parts : p.heads;
    const int head = unit % fast;  // query head; kv head * parts + part
    unit /= fast;
    const int seq = unit % p.n_seqs, slot = unit / p.n_seqs;
    const Span sq = span_of(p.cu_q, seq, p.rows_q, p.max_q), sk = span_of(p.cu_k, seq, p.rows_k, p.max_k);
    const int off = sk.len - sq.len;  // position of query i: i + off
    const int stand_len = KIND == DKV ? sk.len : sq.len, stream_len = KIND == DKV ? sq.len : sk.len;
    const int n_slots = (stand_len + kStand - 1) / kStand;
    if (slot >= n_slots) return;
    // the longest first: late queries see most keys, early keys are seen by most queries
    const int a_first = (KIND == DKV ? slot : n_slots - 1 - slot) * kStand, a_rows = min(kStand, stand_len - a_first);
    const int G = p.heads / p.kv_heads;
    const int kvh = KIND == DKV ? head / p.parts : head / G;
    int h0 = head, h1 = head + 1;  // query heads
    if (KIND == DKV) {
        const int part = head % p.parts, per = (G + p.parts - 1) / p.parts;
        h0 = kvh * G + min(part * per, G);
        h1 = kvh * G + min(part * per + per, G);
    }
    // visible streamed rows of standing row r
    auto visible = [&](int r, int& lo, int& hi) {
        if (KIND == DKV) {
            lo = p.causal ? max(0, r - off) : 0;
            hi = p.chunk > 0 ? (int)min((int64_t)sq.len, ((int64_t)(r / p.chunk) + 1) * p.chunk - off) : sq.len;
        } else {
            const int pos = r + off;
            lo = p.chunk > 0 && pos > 0 ? pos / p.chunk * p.chunk : 0;
            hi = p.causal ? pos + 1 : sk.len;
        }
    };
    int first, last, unused;
    visible(a_first, first, unused);
    visible(a_first + a_rows - 1, unused, last);
    const int tiles_per_head = last > first ? (last - first + kTile - 1) / kTile : 0, tiles = tiles_per_head * (h1 - h0);

    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 128);
            mbar_init(&p_full[i], 128);
            mbar_init(&p_done[i], 1);
        }
        mbar_init(a_full, C::A_SHARED ? 1 : 256);
        mbar_init(all_done, 1);
        fence_mbar_init();
    }
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    if (KIND != FWD) pdl_wait();

    if (warp == 8) {
        if (lane == 0) {
            prefetch_tmap(&p.tm[0]);
            prefetch_tmap(&p.tm[1]);
        }
        __syncwarp();
        const uint32_t ring = smem_u32(smem + C::RING), bar = smem_u32(full);
        auto load = [&](const CUtensorMap* tm, uint32_t dst, int n_heads, int h, int64_t row, uint32_t b, int block) {
#pragma unroll
            for (int i = 0; i < C::BLOCKS; ++i)
                if (n_heads > 1)
                    tma_load_3d_elect(dst + i * block, tm, i * 64, h, (int)row, b);
                else
                    tma_load_2d_elect(dst + i * block, tm, i * 64, (int)row, b);
        };
        if (C::A_SHARED && tiles > 0) {
            const uint32_t a = smem_u32(smem), ab = smem_u32(a_full);
            mbar_arrive_expect_tx_elect(ab, 2 * C::A_TILE);
            load(&p.tmA[0], a, p.kv_heads, kvh, sk.first + a_first, ab, C::A_BLOCK);
            load(&p.tmA[1], a + C::A_TILE, p.kv_heads, kvh, sk.first + a_first, ab, C::A_BLOCK);
        }
        bool ok = true;
        int h = h0, t = 0;
        for (int j = 0; j < tiles && ok; ++j) {
            const int st = j % C::STAGES;
            if (j >= C::STAGES) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (uint32_t)(j / C::STAGES - 1) & 1u, p.status, DEV_ERR_EMPTY_WAIT));
            if (!ok) break;
            const uint32_t b = bar + st * 8, dst = ring + st * C::STAGE;
            mbar_arrive_expect_tx_elect(b, C::STAGE);
            const int64_t row = (KIND == DKV ? sq.first : sk.first) + first + t * kTile;
            const int n_heads = KIND == DKV ? p.heads : p.kv_heads, hh = KIND == DKV ? h : kvh;
            load(&p.tm[0], dst, n_heads, hh, row, b, C::BLOCK);
            load(&p.tm[1], dst + C::TILE, n_heads, hh, row, b, C::BLOCK);
            if (++t == tiles_per_head) {
                t = 0;
                ++h;
            }
        }
    } else if (warp == 9) {
        constexpr uint32_t idesc_s = umma_idesc_bf16(kStand, kTile), idesc_acc = umma_idesc_bf16(kStand, HD) | (1u << 16);  // streamed tile: its K extent in rows
        const uint32_t ring = smem_u32(smem + C::RING);
        const uint64_t a_d = umma_desc_k128(smem_u32(smem)), k_d = umma_desc_k128(ring), n_d = umma_desc_n128(ring, C::BLOCK);
        auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, code)); };
        // S or dP of a tile: standing operand `which` times streamed operand `which`
        auto product = [&](uint32_t d, int which, int st) {
            const uint64_t b = k_d + (uint64_t)(uint32_t)((st * C::STAGE + which * C::TILE) >> 4);
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) {
                const uint64_t bi = b + (i >> 2) * (C::BLOCK >> 4) + 2 * (i & 3);
                if constexpr (C::A_SHARED)
                    umma_bf16_elect(d, a_d + (uint64_t)(uint32_t)((which * C::A_TILE + (i >> 2) * C::A_BLOCK) >> 4) + 2 * (i & 3), bi, idesc_s, i > 0);
                else
                    umma_bf16_ts(d, tmem + (which ? C::A1 : C::A0) + i * 8, bi, idesc_s, i > 0);
            }
        };
        auto accumulate = [&](uint32_t d, uint32_t a, int which, int st, bool more) {
            const uint64_t b = n_d + (uint64_t)(uint32_t)((st * C::STAGE + which * C::TILE) >> 4);
#pragma unroll
            for (int i = 0; i < kTile / 16; ++i) umma_bf16_ts(d, a + i * 8, b + i * 128, idesc_acc, more || i > 0);
        };
        auto scores = [&](int j) {
            const int st = j % C::STAGES;
            if (!wait(&full[st], (uint32_t)(j / C::STAGES) & 1u, DEV_ERR_FULL_WAIT)) return false;
            const int valid = stream_len - first - j % tiles_per_head * kTile;
            if (valid < kTile) {
                // rows behind the sequence weigh zero, but what lies there may not be finite
                for (int i = lane; i < (kTile - valid) * 8 * 2 * C::BLOCKS; i += 32) {
                    const int c = i & 7, b = (i >> 3) % (2 * C::BLOCKS), r = valid + (i >> 3) / (2 * C::BLOCKS);
                    *(uint4*)(smem + C::RING + st * C::STAGE + b * C::BLOCK + r * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }
            tc_fence_after();
            const uint32_t d = tmem + C::S + (j & 1) * C::S_STEP;
            product(d, 0, st);
            if (KIND != FWD) product(d + kTile, 1, st);
            umma_commit_elect(&s_full[j & 1]);
            return true;
        };
        bool ok = tiles > 0 && wait(a_full, 0, DEV_ERR_FULL_WAIT);
        tc_fence_after();
        if (ok) ok = scores(0);
        if (ok && tiles > 1) ok = scores(1);
        for (int j = 0; j < tiles && ok; ++j) {
            const int st = j % C::STAGES, b = j & 1;
            const uint32_t ph = (uint32_t)(j >> 1) & 1u;
            if (KIND == FWD && j + 2 < tiles) {  // S of this tile is in registers: the next one of its group takes its place
                ok = wait(&s_free[b], ph, DEV_ERR_ACC_WAIT) && scores(j + 2);
                if (!ok) break;
            }
            ok = wait(&p_full[b], ph, DEV_ERR_ACC_WAIT);
            if (!ok) break;
            tc_fence_after();
            if constexpr (KIND == FWD) {
                accumulate(tmem + C::ACC + b * HD, tmem + C::P + b * (kTile / 2), 1, st, j > 1);
                umma_commit_elect(&p_done[b]);
            } else if constexpr (KIND == DQ) {
                accumulate(tmem + C::ACC, tmem + C::S + b * C::S_STEP, 0, st, j > 0);
            } else {
                accumulate(tmem + C::ACC + HD, tmem + C::S + b * C::S_STEP, 1, st, j > 0);      // dV
                accumulate(tmem + C::ACC, tmem + C::S + b * C::S_STEP + kTile, 0, st, j > 0);   // dK
            }
            umma_commit_elect(&empty[st]);
            if (KIND != FWD && j + 2 < tiles) ok = scores(j + 2);  // behind the products that read this buffer
        }
        if (ok && tiles > 0) umma_commit_elect(all_done);
    } else {
        const int group = warp / kWarpsOfGroup, r = tid % kStand;
        const uint32_t lanes = (uint32_t)((warp % kWarpsOfGroup) * 32) << 16;
        const bool live = r < a_rows;
        const int row = a_first + r;
        const int64_t grow = (KIND == DKV ? sk.first : sq.first) + row;  // row of the buffers
        const int a_head = KIND == DKV ? kvh : head;
        bool ok = true;
        if (!C::A_SHARED && tiles > 0) {
            if (group == 0 || KIND != FWD) {
                const bf16* src = group == 0 ? p.a0 + grow * p.a0_stride : p.a1 + grow * p.a1_stride;
                row_to_tmem<HD>(tmem + lanes + (group == 0 ? C::A0 : C::A1), live ? src + (int64_t)a_head * p.hd : nullptr, p.hd);
            }
            tc_fence_before();
            mbar_arrive(a_full);
        }
        int lo = 0, hi = 0;
        if (live) visible(row, lo, hi);
        float2* const stats = (float2*)(smem + C::ROWS);
        float m = -INFINITY, sum = 0.f, lse2 = 0.f, dd = 0.f;
        if (KIND == DQ && live) {
            const float l = p.lse[(int64_t)head * p.rows_q + grow];
            lse2 = l == -INFINITY ? 0.f : l * kLog2e;
            dd = p.d[(int64_t)head * p.rows_q + grow];
        }
        // lse (first half of the group) and D (second half) of a streamed query
        auto fetch = [&](int j) {
            if (j >= tiles) return 0.f;
            const int col = first + j % tiles_per_head * kTile + (r & 63), h = h0 + j / tiles_per_head;
            if (col >= sq.len) return 0.f;
            const float v = __ldg((r < 64 ? p.lse : p.d) + (int64_t)h * p.rows_q + sq.first + col);
            return r < 64 ? (v == -INFINITY ? 0.f : v * kLog2e) : v;
        };
        float ahead = KIND == DKV ? fetch(group) : 0.f;
        // A wait that ran out lets the warp go on without waiting, since the others of its group wait for it at their barrier.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, p.status, DEV_ERR_ACC_WAIT));
        };
        for (int j = group; j < tiles; j += 2) {
            const int b = group;
            const uint32_t ph = (uint32_t)(j >> 1) & 1u;
            const uint32_t buf = tmem + lanes + C::S + b * C::S_STEP;
            const int base = first + j % tiles_per_head * kTile;
            const int c_lo = lo - base, c_hi = hi - base;  // visible columns
            const bool whole = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= kTile);
            float2* const q_stats = stats + (b * 2 + (int)ph) * kTile;
            if (KIND == DKV) {
                ((float*)(q_stats + (r & 63)))[r < 64 ? 0 : 1] = ahead;
                ahead = fetch(j + 2);
                group_barrier(group);
            }
            wait(&s_full[b], ph);
            tc_fence_after();
            if constexpr (KIND == FWD) {
                uint32_t s[4][16];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld16(buf + k * 16, s[k]);
                tc_wait_ld();
                tc_fence_before();
                mbar_arrive(&s_free[b]);
                if (!whole)
#pragma unroll
                    for (int i = 0; i < kTile; ++i)
                        if (i < c_lo || i >= c_hi) s[i >> 4][i & 15] = 0xff800000u;
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < kTile; ++i) top = fmaxf(top, __uint_as_float(s[i >> 4][i & 15]));
                top *= p.scale_log2;  // positive scale: the maximum stays the maximum
                float corr = 1.f;
                bool moved = false;
                if (top > m + 8.f || m == -INFINITY) {  // the reference moves only when it would be passed by more than 2^8
                    corr = m == -INFINITY ? 0.f : exp2_fast(m - top);
                    moved = m != -INFINITY;
                    m = top;
                }
                const float ref = m == -INFINITY ? 0.f : m;  // nothing visible yet: every weight is zero
                sum *= corr;
                uint32_t w[2][16];
                float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < kTile; i += 2) {
                    const float x = exp2_fast(fmaf(__uint_as_float(s[i >> 4][i & 15]), p.scale_log2, -ref));
                    const float y = exp2_fast(fmaf(__uint_as_float(s[i >> 4][(i & 15) + 1]), p.scale_log2, -ref));
                    part[i >> 1 & 3] += x + y;
                    w[i >> 5][(i & 31) >> 1] = pack2(x, y);
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
                if (j > 1) {  // the product that read the last P, and wrote O
                    wait(&p_done[b], ((uint32_t)(j >> 1) - 1u) & 1u);
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, moved)) {
                    const uint32_t o_at = tmem + lanes + C::ACC + b * HD;
#pragma unroll 1
                    for (int k = 0; k < HD / 16; ++k) {
                        uint32_t o[16];
                        tmem_ld16(o_at + k * 16, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmem_st16(o_at + k * 16, o);
                    }
                }
                tmem_st16(tmem + lanes + C::P + b * (kTile / 2), w[0]);
                tmem_st16(tmem + lanes + C::P + b * (kTile / 2) + 16, w[1]);
            } else {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t s[2][16], dp[2][16], w[16], v[16];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        tmem_ld16(buf + half * 32 + k * 16, s[k]);
                        tmem_ld16(buf + kTile + half * 32 + k * 16, dp[k]);
                    }
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float pr[2], ds[2];
                        float4 st4;
                        if constexpr (KIND == DKV) st4 = *(const float4*)(q_stats + half * 32 + i);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int c = half * 32 + i + e;
                            const float l = KIND == DKV ? (e ? st4.z : st4.x) : lse2, dr = KIND == DKV ? (e ? st4.w : st4.y) : dd;
                            float x = exp2_fast(fmaf(__uint_as_float(s[i >> 4][(i & 15) + e]), p.scale_log2, -l));
                            if (!whole && (c < c_lo || c >= c_hi)) x = 0.f;
                            pr[e] = x;
                            ds[e] = x * (__uint_as_float(dp[i >> 4][(i & 15) + e]) - dr);
                        }
                        w[i >> 1] = pack2(pr[0], pr[1]);
                        v[i >> 1] = pack2(ds[0], ds[1]);
                    }
                    if constexpr (KIND == DKV) {
                        tmem_st16(buf + half * 16, w);
                        tmem_st16(buf + kTile + half * 16, v);
                    } else {
                        tmem_st16(buf + half * 16, v);
                    }
                }
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[b]);
        }
        // ---- results
        if (tiles > 0) wait(all_done, 0);
        tc_fence_after();
        float w0 = tiles > 0 ? 1.f : 0.f, w1 = 0.f;  // weights of the accumulators
        if constexpr (KIND == FWD) {
            stats[group * kStand + r] = make_float2(m, sum);
            groups_barrier();
            const float2 x = stats[r], y = stats[kStand + r];
            const float top = fmaxf(x.x, y.x);
            const float e0 = x.x == -INFINITY ? 0.f : exp2_fast(x.x - top), e1 = y.x == -INFINITY ? 0.f : exp2_fast(y.x - top);
            const float total = fmaf(x.y, e0, y.y * e1);
            w0 = total > 0.f ? e0 / total : 0.f;
            w1 = total > 0.f ? e1 / total : 0.f;
            if (group == 0 && live && p.lse) p.lse[(int64_t)head * p.rows_q + grow] = total > 0.f ? (top + log2f(total)) / kLog2e : -INFINITY;
        } else {
            w0 *= KIND == DQ || group == 0 ? p.scale : 1.f;
        }
        // FWD, DQ: a group stores half of the columns; DKV: dK, dV
        constexpr int WIDTH = KIND == DKV ? HD : HD / 2;
        const int col0 = KIND == DKV ? 0 : group * WIDTH;
        const uint32_t acc = tmem + lanes + C::ACC + (KIND == DKV ? group * HD : col0);
        bf16* const dst = KIND == DKV && group == 1 ? p.out1 + grow * p.out1_stride : p.out0 + grow * p.out0_stride;
        float* const part = KIND == DKV && p.partial
                                ? p.partial + ((((int64_t)group * p.parts + head % p.parts) * p.rows_k + grow) * p.kv_heads + kvh) * p.hd
                                : nullptr;
#pragma unroll 1
        for (int k = 0; k < WIDTH / 16; ++k) {
            float v[16];
            uint32_t o[16], o2[16];
            if (tiles > 0) tmem_ld16(acc + k * 16, o);
            if (KIND == FWD && tiles > 1) tmem_ld16(acc + HD + k * 16, o2);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                v[i] = tiles > 0 ? __uint_as_float(o[i]) * w0 : 0.f;
                if (KIND == FWD && tiles > 1) v[i] = fmaf(__uint_as_float(o2[i]), w1, v[i]);
            }
            const int c = col0 + k * 16;
#pragma unroll
            for (int i = 0; i < 16; i += 8)
                if (live && c + i < p.hd) {
                    if (KIND == DKV && part) {
                        *(float4*)(part + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        *(float4*)(part + c + i + 4) = make_float4(v[i + 4], v[i + 5], v[i + 6], v[i + 7]);
                    } else {
                        *(uint4*)(dst + (int64_t)a_head * p.hd + c + i) =
                            make_uint4(pack2(v[i], v[i + 1]), pack2(v[i + 2], v[i + 3]), pack2(v[i + 4], v[i + 5]), pack2(v[i + 6], v[i + 7]));
                    }
                }
            __syncwarp();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 512);
}

// D[h][row] = sum of dO o O over the head: L = HD / 8 lanes a row, neighbouring rows in neighbouring lanes
template <int L>
__global__ void __launch_bounds__(256) k_attn_dot(const bf16* __restrict__ d_out, const bf16* __restrict__ out, int64_t stride, const int* cu_q, int n_seqs, int64_t rows, int heads,
                                                  int hd, float* __restrict__ d) {
    pdl_launch_dependents();
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int h = blockIdx.y, c = threadIdx.x % L * 8;
    const bool live = row < rows && row >= cu_q[0] && row < cu_q[n_seqs];
    float a = 0.f;
    if (live && c < hd) {
        const uint4 x = __ldg((const uint4*)(d_out + row * stride + (int64_t)h * hd + c)), y = __ldg((const uint4*)(out + row * stride + (int64_t)h * hd + c));
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a = fmaf(bf16_lo(xs[i]), bf16_lo(ys[i]), a);
            a = fmaf(bf16_hi(xs[i]), bf16_hi(ys[i]), a);
        }
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (live && c == 0) d[(int64_t)h * rows + row] = a;
}

// dK and dV from the parts of the query heads, added in their order
__global__ void __launch_bounds__(256) k_attn_join(const float* __restrict__ partial, int parts, const int* cu_k, int n_seqs, int64_t rows, int kv_heads, int hd, bf16* dk,
                                                   int64_t dk_stride, bf16* dv, int64_t dv_stride) {
    pdl_wait();
    const int per_row = kv_heads * hd / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / per_row;
    if (row >= rows || row < cu_k[0] || row >= cu_k[n_seqs]) return;
    const int c = (int)(i % per_row) * 4;
    const int64_t plane = rows * kv_heads * hd;
    const float* src = partial + (int64_t)blockIdx.y * parts * plane + row * kv_heads * hd + c;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < parts; ++q) {
        const float4 v = __ldg((const float4*)(src + q * plane));
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
    }
    bf16* dst = blockIdx.y ? dv + row * dv_stride : dk + row * dk_stride;
    *(uint2*)(dst + c) = make_uint2(pack2(a.x, a.y), pack2(a.z, a.w));
}

template <int HD, int KIND>
int run(const Dev& p, int64_t blocks, cudaStream_t s, bool pdl) {
    using C = Cfg<HD, KIND>;
    const cudaError_t e = allow_shared<k_train_attn<HD, KIND>>(C::SMEM);
    if (e != cudaSuccess) return (int)e;
    if (blocks > INT32_MAX) return (int)cudaErrorInvalidValue;
    return (int)launch_k(k_train_attn<HD, KIND>, dim3((unsigned)blocks), dim3(kThreads), (size_t)C::SMEM, s, pdl, p);
}

Dev common(const AttnCall& c) {
    Dev p;
    memset(&p, 0, sizeof p);
    p.cu_q = c.cu_q;
    p.cu_k = c.cu_k;
    p.rows_q = c.rows_q;
    p.rows_k = c.rows_k;
    p.max_q = c.max_q;
    p.max_k = c.max_k;
    p.n_seqs = c.n_seqs;
    p.heads = c.heads;
    p.kv_heads = c.kv_heads;
    p.hd = c.hd;
    p.causal = c.causal;
    p.chunk = c.chunk;
    p.parts = 1;
    p.scale = c.scale;
    p.scale_log2 = c.scale * kLog2e;
    p.lse = c.lse;
    p.status = c.status;
    return p;
}

bool map_heads(CUtensorMap* tm, const bf16* x, int64_t rows, int64_t stride, int heads, int hd, int box) {
    return make_tmap_2d(nullptr, tm, x, (uint64_t)rows, (uint64_t)hd, (uint64_t)stride, (uint32_t)box, (uint32_t)heads, (uint32_t)hd);
}

int64_t blocks_for(const AttnCall& c, int most, int fast) { return (int64_t)((most + kStand - 1) / kStand) * c.n_seqs * fast; }

// Blocks of dK, dV by query heads: one block adds all heads of its kv head up where that gives each of the 148 SMs two blocks to even out
// unequal lengths; else the heads are dealt to as many blocks as that takes, and their sums are joined through the workspace.
int parts_of(const AttnCall& c) {
    const int G = c.heads / c.kv_heads;
    const int64_t blocks = blocks_for(c, c.max_k, c.kv_heads);
    int parts = 1;
    while (parts < G && blocks * parts < 2 * 148) ++parts;
    const int per = (G + parts - 1) / parts;
    return (G + per - 1) / per;
}

}  // namespace

int64_t attention_workspace_bytes(const AttnCall& c) {
    const int64_t d = ((int64_t)c.heads * c.rows_q * 4 + 255) / 256 * 256;
    const int parts = parts_of(c);
    return d + (parts > 1 ? 2 * parts * c.rows_k * c.kv_heads * c.hd * 4 : 0);
}

int launch_attention_train_forward(const AttnCall& c, cudaStream_t s) {
    if (c.n_seqs == 0 || c.max_q == 0 || c.rows_q == 0) return 0;
    Dev p = common(c);
    // no keys at all: any valid map, none of its rows is read
    if (!map_heads(&p.tm[0], c.rows_k ? c.k : c.q, c.rows_k ? c.rows_k : c.rows_q, c.rows_k ? c.k_stride : c.q_stride, c.kv_heads, c.hd, kTile)) return -1000;
    if (!map_heads(&p.tm[1], c.rows_k ? c.v : c.q, c.rows_k ? c.rows_k : c.rows_q, c.rows_k ? c.v_stride : c.q_stride, c.kv_heads, c.hd, kTile)) return -1000;
    p.a0 = c.q;
    p.a0_stride = c.q_stride;
    p.out0 = c.out;
    p.out0_stride = c.out_stride;
    const int64_t blocks = blocks_for(c, c.max_q, c.heads);
    return c.hd <= 64 ? run<64, FWD>(p, blocks, s, false) : run<128, FWD>(p, blocks, s, false);
}

int launch_attention_train_backward(const AttnCall& c, cudaStream_t s) {
    const bool queries = c.max_q > 0 && c.rows_q > 0, keys = c.max_k > 0 && c.rows_k > 0;
    if (c.n_seqs == 0 || (!queries && !keys)) return 0;
    float* const d = (float*)c.workspace;
    int rc = 0;
    if (queries) {
        const int lanes = c.hd <= 64 ? 8 : 16;
        const dim3 grid((unsigned)((c.rows_q + 256 / lanes - 1) / (256 / lanes)), (unsigned)c.heads);
        rc = lanes == 8 ? (int)launch_k(k_attn_dot<8>, grid, dim3(256), 0, s, false, c.d_out, c.out, c.out_stride, c.cu_q, c.n_seqs, c.rows_q, c.heads, c.hd, d)
                        : (int)launch_k(k_attn_dot<16>, grid, dim3(256), 0, s, false, c.d_out, c.out, c.out_stride, c.cu_q, c.n_seqs, c.rows_q, c.heads, c.hd, d);
        if (rc) return rc;
    }
    if (keys) {
        Dev p = common(c);
        const bf16 *q = queries ? c.q : c.k, *g = queries ? c.d_out : c.k;  // no queries: any valid map, none of its rows is read
        const int64_t rows = queries ? c.rows_q : c.rows_k;
        if (!map_heads(&p.tm[0], q, rows, queries ? c.q_stride : c.k_stride, queries ? c.heads : c.kv_heads, c.hd, kTile)) return -1000;
        if (!map_heads(&p.tm[1], g, rows, queries ? c.out_stride : c.k_stride, queries ? c.heads : c.kv_heads, c.hd, kTile)) return -1000;
        if (!map_heads(&p.tmA[0], c.k, c.rows_k, c.k_stride, c.kv_heads, c.hd, kStand)) return -1000;
        if (!map_heads(&p.tmA[1], c.v, c.rows_k, c.v_stride, c.kv_heads, c.hd, kStand)) return -1000;
        p.a0 = c.k;
        p.a0_stride = c.k_stride;
        p.a1 = c.v;
        p.a1_stride = c.v_stride;
        p.d = d;
        p.parts = parts_of(c);
        p.partial = p.parts > 1 ? (float*)((char*)c.workspace + ((int64_t)c.heads * c.rows_q * 4 + 255) / 256 * 256) : nullptr;
        p.out0 = c.dk;
        p.out0_stride = c.k_stride;
        p.out1 = c.dv;
        p.out1_stride = c.v_stride;
        const int64_t blocks = blocks_for(c, c.max_k, c.kv_heads * p.parts);
        rc = c.hd <= 64 ? run<64, DKV>(p, blocks, s, false) : run<128, DKV>(p, blocks, s, false);
        if (rc) return rc;
        if (p.partial) {
            const int64_t vecs = c.rows_k * c.kv_heads * c.hd / 4;
            rc = (int)launch_k(k_attn_join, dim3((unsigned)((vecs + 255) / 256), 2), dim3(256), 0, s, false, (const float*)p.partial, p.parts, c.cu_k, c.n_seqs, c.rows_k, c.kv_heads,
                               c.hd, c.dk, c.k_stride, c.dv, c.v_stride);
            if (rc) return rc;
        }
    }
    if (queries) {
        Dev p = common(c);
        if (!map_heads(&p.tm[0], keys ? c.k : c.q, keys ? c.rows_k : c.rows_q, keys ? c.k_stride : c.q_stride, c.kv_heads, c.hd, kTile)) return -1000;
        if (!map_heads(&p.tm[1], keys ? c.v : c.q, keys ? c.rows_k : c.rows_q, keys ? c.v_stride : c.q_stride, c.kv_heads, c.hd, kTile)) return -1000;
        p.a0 = c.q;
        p.a0_stride = c.q_stride;
        p.a1 = c.d_out;
        p.a1_stride = c.out_stride;
        p.d = d;
        p.out0 = c.dq;
        p.out0_stride = c.q_stride;
        const int64_t blocks = blocks_for(c, c.max_q, c.heads);
        rc = c.hd <= 64 ? run<64, DQ>(p, blocks, s, false) : run<128, DQ>(p, blocks, s, false);
    }
    return rc;
}

}  // namespace tffn
