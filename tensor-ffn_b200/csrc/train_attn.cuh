// What the forward and backward kernels of training attention (train_attn.cu, train_attn_bwd.cu) share: the call as the device sees it,
// which rows a block computes and which it can see, and small helpers.
#pragma once
#include "launch.h"
#include "pair.cuh"
#include "ptx.cuh"
#include "train.h"

namespace tffn {

constexpr int kStand = 128;  // rows that stand still: queries for O and dQ, keys for dK and dV
constexpr float kLog2e = 1.4426950408889634f;

// n / d for 0 <= n < 2^31 by a multiplication: with 2^(l - 1) < d <= 2^l, m = ceil(2^(31 + l) / d) < 2^32
struct FastDiv {
    uint32_t d, m, s;
    __host__ static FastDiv of(int64_t d) {
        FastDiv f;
        int l = 0;
        while ((int64_t)1 << l < d) ++l;
        f.d = (uint32_t)d;
        f.s = 31 + l;
        f.m = (uint32_t)((((uint64_t)1 << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d);
        return f;
    }
    __device__ __forceinline__ int div(int n) const { return (int)(((uint64_t)(uint32_t)n * m) >> s); }
};

struct AttnDev {
    CUtensorMap tm[2];   // streamed operands: K, V or Q, dO; boxes of rows x 64 columns of one head
    CUtensorMap tmA[2];  // standing operands, boxes of 128 rows
    const int *cu_q, *cu_k;
    int64_t rows_q, rows_k;
    int max_q, max_k, n_seqs, heads, kv_heads, group, hd, causal, chunk;  // group: query heads of a kv head
    FastDiv by_fast, by_group, by_parts, by_chunk;                        // by_fast: units of a slot of a sequence
    int chunk_slots;     // of a chunk, or 0
    int most_levels;     // that the units of all sequences are looked at on: AttnWalk
    int units;           // of the call, at most: below 2^30, so that sums over units stay in 32 bits whatever the offsets say
    int parts;           // units that a block takes at once (forward); parts of the query heads of a kv head (dK, dV)
    float scale, scale_log2;
    float* lse;          // [heads][rows_q]
    float* d;            // [heads][rows_q]
    bf16 *out0, *out1;   // O; dQ; dK, dV
    int64_t out0_stride, out1_stride;
    float* partial;      // parts > 1: dK, dV as fp32 [2][parts][rows_k][kv_heads][hd]
    int* status;
};

// rows of a sequence, whatever the offsets say inside the buffer and not longer than promised
struct AttnSpan {
    int first, len;
};
__device__ __forceinline__ AttnSpan attn_span(int begin, int end, int64_t rows, int most) {
    const int b = min(max(begin, 0), (int)rows), e = min(max(end, b), (int)rows);
    return {b, min(e - b, most)};
}

// visible streamed rows [lo, hi) of standing row r: of a query, or of a key (DKV)
template <bool DKV>
__device__ __forceinline__ void attn_visible(const AttnDev& p, int q_len, int k_len, int r, int& lo, int& hi) {
    const int off = k_len - q_len;  // position of query i: i + off
    if (DKV) {
        lo = p.causal ? max(0, r - off) : 0;
        hi = p.chunk > 0 ? (int)min((int64_t)q_len, ((int64_t)p.by_chunk.div(r) + 1) * p.chunk - off) : q_len;
    } else {
        const int pos = r + off;
        lo = p.chunk > 0 && pos > 0 ? p.by_chunk.div(pos) * p.chunk : 0;
        hi = p.causal ? pos + 1 : k_len;
    }
}

// bits [lo, hi) of 64, whatever lo and hi
__device__ __forceinline__ uint64_t bits_between(int lo, int hi) {
    const int from = min(max(lo, 0), 64), to = min(max(hi, 0), 64);
    return (to == 64 ? ~0ull : (1ull << to) - 1) & ~(from == 64 ? ~0ull : (1ull << from) - 1);
}

// Which units a block computes. A unit is (fast, sequence, slot): `slots_of` says how many slots a sequence has, and heads are fastest, so that blocks
// that stream the same rows run together. The units that there are, empty ones not counted, stand in one order, longest first: by `level`, which is how
// much of the other side a slot sees (its distance from the sequence's first block, or in a chunk from the chunk's), and then by sequence.
// A block has one of every round of `grid` units, in every other round counted from the end, so that the blocks end together.
// 1 x 8 192, 28 heads of 128, forward: 411 us, with rounds counted from the start 469; 32 ragged x 512, 14 heads of 64, backward 80 us, else 112.
//
// A look at 32 sequences at one level costs 0.2 us, and all of them at every level is sequences x longest: one of 8 192 among 4 095 of 64 would be 1.3 ms of
// looking (and a million of them long enough for the waits of the others to run out). Where that is more than four looks a unit, each 32 sequences are in
// that order by themselves, one after the other, which is as many looks as there are units at most (those 4 096: forward 0.29 ms).
struct AttnUnit {
    int fast, slot;
    AttnSpan q, k;
};
struct AttnWalk {
    bool apart = false;                               // each 32 sequences by themselves
    int levels = -1, period, turns;                   // levels = period * turns: by place in a chunk and then by chunk, or by place in the sequence (one turn)
    int round = 0, level = 0, first = 0, before = 0;  // first: of 32 sequences; before: units in front of these of this level
    int loaded = -1, slots = 0, phase = 0;            // the lane's sequence, of those from `loaded` on
    AttnSpan q = {0, 0}, k = {0, 0};
};
// the block's next unit, for a whole warp: lane = sequence
template <bool DKV, typename F>
__device__ __forceinline__ bool next_unit(const AttnDev& p, AttnWalk& at, AttnUnit& u, F&& slots_of) {
    const int grid = gridDim.x, lane = threadIdx.x & 31;
    const int target = at.round * grid + (at.round & 1 ? grid - 1 - (int)blockIdx.x : (int)blockIdx.x);
    if (target >= p.units) return false;
    auto load = [&](int first) {
        const int seq = first + lane;
        at.loaded = first;
        at.q = at.k = {0, 0};
        if (seq < p.n_seqs) {
            at.q = attn_span(p.cu_q[seq], p.cu_q[seq + 1], p.rows_q, p.max_q);
            at.k = attn_span(p.cu_k[seq], p.cu_k[seq + 1], p.rows_k, p.max_k);
        }
        at.slots = slots_of(DKV ? at.k.len : at.q.len);
        at.phase = 0;  // of the first query in its chunk, rounded down, so that the slots that see the end of one chunk and the start of the next come first
        if (!DKV && p.chunk_slots > 0) {
            const int off = max(at.k.len - at.q.len, 0);
            at.phase = min(slots_of((off - p.by_chunk.div(off) * p.chunk) / kStand * kStand), p.chunk_slots);
        }
    };
    auto measure = [&](int most) {
        most = __reduce_max_sync(0xffffffffu, most);
        const bool by_chunk = p.chunk_slots > 0 && p.chunk_slots < most;
        at.period = by_chunk ? p.chunk_slots : most;
        // queries may begin in the middle of a chunk, so that they touch one more
        at.turns = !by_chunk ? 1 : (most + at.period - 1) / at.period + (DKV ? 0 : 1);
        at.levels = at.period * at.turns;
    };
    if (at.levels < 0) {  // how long the longest sequence is: the call's bounds may be far above it
        int most = 0;
#pragma unroll 1
        for (int first = 0; first < p.n_seqs; first += 32) {
            load(first);
            most = max(most, at.slots);
        }
        measure(most);
        at.apart = at.levels > p.most_levels;
        if (at.apart) {
            load(0);
            measure(at.slots);
        }
    }
#pragma unroll 1
    for (;;) {
        if (at.level >= at.levels) {
            at.first += 32;
            if (!at.apart || at.first >= p.n_seqs) return false;
            load(at.first);
            measure(at.slots);
            at.level = 0;
            continue;
        }
        const bool by_chunk = at.turns > 1;
        if (at.loaded != at.first) load(at.first);
        // at most one slot of a sequence is at a level: this, unless it is negative or more than there are
        auto slot_at = [&](int pos, int turn, int slots, int phase) {
            return DKV && by_chunk ? turn * at.period + pos : slots - 1 - (turn * at.period + at.period - 1 - pos - (by_chunk ? phase : 0));
        };
        if (p.n_seqs <= 32 && p.n_seqs * p.n_seqs * (int64_t)p.by_fast.d < 3 * grid) {  // few units a level: 32 levels at a time, lane = level
            const int level = at.level + lane, pos = by_chunk ? level / at.turns : level, turn = level - pos * at.turns;
            int sum = 0;
#pragma unroll 1
            for (int i = 0; i < p.n_seqs; ++i) {
                const int slots = __shfl_sync(0xffffffffu, at.slots, i), slot = slot_at(pos, turn, slots, __shfl_sync(0xffffffffu, at.phase, i));
                sum += slot >= 0 && slot < slots && level < at.levels;
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned reach = __ballot_sync(0xffffffffu, sum > p.by_fast.div(target - at.before));
            const int skip = reach ? __ffs(reach) - 1 : 32;
            if (skip > 0) {
                at.before += __shfl_sync(0xffffffffu, sum, skip - 1) * (int)p.by_fast.d;
                at.level += skip;
            }
            if (!reach) continue;
        }
        const int pos = by_chunk ? at.level / at.turns : at.level, slot = slot_at(pos, at.level - pos * at.turns, at.slots, at.phase);
        const bool there = slot >= 0 && slot < at.slots;
        const unsigned all = __ballot_sync(0xffffffffu, there);
        const int rest = target - at.before, rank = p.by_fast.div(rest);
        if (rank < __popc(all)) {
            const int from = __ffs(__ballot_sync(0xffffffffu, there && __popc(all & ((1u << lane) - 1u)) == rank)) - 1;
            u.fast = rest - rank * (int)p.by_fast.d;
            u.slot = __shfl_sync(0xffffffffu, slot, from);
            u.q.first = __shfl_sync(0xffffffffu, at.q.first, from);
            u.q.len = __shfl_sync(0xffffffffu, at.q.len, from);
            u.k.first = __shfl_sync(0xffffffffu, at.k.first, from);
            u.k.len = __shfl_sync(0xffffffffu, at.k.len, from);
            ++at.round;
            return true;
        }
        at.before += __popc(all) * (int)p.by_fast.d;
        if (at.apart) {
            ++at.level;
            continue;
        }
        at.first += 32;
        if (at.first >= p.n_seqs) {
            at.first = 0;
            ++at.level;
        }
    }
}

// What one warp has worked out of a unit reaches the others through a few slots of shared memory, each with a barrier for the warps that read it
// and one for the warp that fills it. A slot is free again when every reader has copied it.
constexpr int kUnitSlots = 4;

// boxes of 64 columns of `rows` rows of one head, block bytes apart in shared memory
template <int BLOCKS>
__device__ __forceinline__ void load_head(const CUtensorMap* tm, uint32_t dst, int block, int n_heads, int head, int row, uint32_t bar) {
#pragma unroll
    for (int i = 0; i < BLOCKS; ++i)
        if (n_heads > 1)
            tma_load_3d_elect(dst + i * block, tm, i * 64, head, row, bar);
        else
            tma_load_2d_elect(dst + i * block, tm, i * 64, row, bar);
}
// Zeros in rows [valid, rows) of `blocks` blocks of 128-byte rows, by a whole warp: rows behind a sequence weigh zero, but what lies there
// may not be finite. A tile that several groups' products read is zeroed by each of them: the same zeros, whenever the
// others' products read them.
__device__ __forceinline__ void zero_rows(uint8_t* at, int block, int blocks, int valid, int rows) {
    for (int i = threadIdx.x & 31; i < (rows - valid) * 8 * blocks; i += 32) {
        const int c = i & 7, b = (i >> 3) % blocks, r = valid + (i >> 3) / blocks;
        *(uint4*)(at + b * block + r * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
    __syncwarp();
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x of two values below 127 on the FMA pipe: x = n + f with |f| <= 1/2, 2^f by a polynomial of degree 4 fitted for the least largest
// relative error (2.7e-6, Remez exchange), n added to its exponent. Values below -126 give 2^-126.
__device__ __forceinline__ F2 exp2_poly(F2 x) {
    float a, b;
    split2(x, a, b);
    x = f2(fmaxf(a, -126.f), fmaxf(b, -126.f));
    const float big = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, which is then the low bits
    const F2 t = add2(x, f2(big, big)), f = fma2(add2(t, f2(-big, -big)), f2(-1.f, -1.f), x);
    F2 y = f2(0.009570102207362652f, 0.009570102207362652f);
    y = fma2(y, f, f2(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, f, f2(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, f, f2(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, f, f2(0.9999992847442627f, 0.9999992847442627f));
    float ya, yb, ta, tb;
    split2(y, ya, yb);
    split2(t, ta, tb);
    return f2(__int_as_float(__float_as_int(ya) + (__float_as_int(ta) << 23)), __int_as_float(__float_as_int(yb) + (__float_as_int(tb) << 23)));
}

// 64 bytes of each of a warp's 32 rows (lane = row) to rows `row_bytes` apart: through 2 KB of shared memory, so that four lanes write a row's
// 64 bytes and no sector is written in halves. `rows` rows and `pieces` of 16 bytes are written.
__device__ __forceinline__ void store_rows(uint8_t* mine, const uint4 (&v)[4], char* to, int64_t row_bytes, int rows, int pieces) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) *(uint4*)(mine + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4)) = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2), c = lane & 3;
        const uint4 x = *(const uint4*)(mine + r * 64 + ((c ^ (r >> 1 & 3)) << 4));
        if (r < rows && c < pieces) *(uint4*)(to + r * row_bytes + c * 16) = x;
    }
    __syncwarp();
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}

// host side (train_attn.cu)
// units of a launch, its grid, and how many levels all sequences are looked at on
unsigned set_units(AttnDev& p, int64_t units, int num_sms);
constexpr int64_t kMostUnits = 1 << 30;
// blocks of kStand rows that sequences of at most `most` rows can have, out of `rows`: each one's last block may be the only one that is not full
int64_t blocks_of_rows(const AttnCall& c, int most, int64_t rows);
AttnDev attn_dev(const AttnCall& c);
bool map_heads(CUtensorMap* tm, const bf16* x, int64_t rows, int64_t stride, int heads, int hd, int box);

}  // namespace tffn
