// Backward pass of the attention of packed training sequences on the tensor cores. With P = exp(scale Q K^T - lse) inside the mask and 0
// outside (formed again from lse: nothing of the size queries x keys is ever stored), dP = dO V^T and D = rowsum(P o dP):
//   dS = P o (dP - D),   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO
//
// Two kernels of one shape, one after the other. 128 rows stand still in shared memory while tiles of 64 rows of the other side stream past:
//   k<DQ>   S = Q K^T,   dP = dO V^T     | dQ += dS K,    M += P K
//   k<DKV>  S^T = K Q^T, dP^T = V dO^T   | dK += dS^T Q,  dV += P^T dO
// The left products take both operands along the head from shared memory; the right ones take the streamed tile a second time, read the
// other way round, and P or dS from the tensor memory that S or dP came from.
//
// D. rowsum(dO o O) with O as it was stored is off by up to 2^-8 of each term, and where a row sees few keys dP - D cancels: two keys of which
// one has all the weight leave 3% in dQ. So k<DQ> starts from that D', sums dS' = P o (dP - D') over the row in fp32, which is D - D', and
// takes dQ = scale (sum dS' K - (D - D') sum P K); the exact D goes back to memory for k<DKV>. It costs the product P K, a fourth one.
//
// Rounding: P and dS enter their products as bf16 (half a step, as inputs and results have), everything else is fp32 until it is stored.
// Every output row has one block that adds it up in one order: no atomics, the same bits on every run. That is why dQ is not added up by the blocks
// of dK, dV: 8 products of a tile instead of 5 (6 with the exact D), but no sum of dQ through memory.
//
// A persistent block of three (64 columns a head) or two (128) groups of four warps, thread = standing row, so that a row's mask is an interval of
// columns; the groups take turns at the tiles, one's exponentials under the others' products. Four more warps turn the accumulators into results
// while the groups are at the next unit. One warp works out the units and fills the rings by TMA; one per group issues its products.
// The sums of all tiles go to the same accumulators: the product warps take turns at them, each waiting for the one before, so that a row
// is always added up in one order.
//
// All these programs run at once, and short sequences go through all of their code all the time: what does not fit the instruction cache
// is what such a call waits for (32 ragged sequences of up to 512 queries, 14 / 2 heads of 64 columns: 112 us; with a variant of P for masks and
// unrolled waits 157 us, and then with the results in the groups' hands 152 us).
//
// What bounds it: 128 columns: the products, 1 280 cycles a tile, of which the left ones wait for shared memory, where both of their operands are
// (1 x 8 192, 28 / 4 heads: 1 640 us in a row of calls, 0.74 PFLOP/s counted as the five products that there have to be, 1.2 as the eight that are
// formed, under the power limit; 1 430 to 1 500 in calls by the dozen with pauses between); 64 columns: 640 cycles of products, 512 of exponentials and
// as many of fp32 arithmetic in about 900 (8 x 4 096, 14 / 2 heads: 890 us, 0.68; in a row of calls 1 040); short sequences: the chain S, P, dP, dS, product of a unit of few
// tiles, and the calls around (the 32 sequences above, with the order of units of now and all heads of a kv head in one block: 73 us, of which dot
// products 10; 77 on inputs that change from call to call).
#include "train_attn.cuh"
#include <algorithm>
#include <cstring>
#include <type_traits>

namespace tffn {

namespace {

constexpr int kTile = 64;

// registers of a thread of this warp and its three neighbours from here on; all four come here
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// 128 standing rows of one head (of one kv head and some of its query heads for dK, dV) and the streamed rows that any of them sees
struct Unit {
    int q_first, k_first, q_len, k_len;
    int a_first, a_rows;  // standing rows within the sequence
    int head, kvh, part;  // standing head: of the queries, or of the keys
    int h0, h1;           // query heads
    int first;            // first streamed row within the sequence
    int tiles_per_head, tiles;  // tiles = -1: no more work
};
template <bool DKV>
__device__ __forceinline__ void unit_of(const AttnDev& p, const AttnUnit& u, Unit& w) {
    w.q_first = u.q.first;
    w.k_first = u.k.first;
    w.q_len = u.q.len;
    w.k_len = u.k.len;
    const int len = DKV ? u.k.len : u.q.len, slots = (len + kStand - 1) / kStand;
    // the longest first: late queries see most keys, early keys are seen by most queries
    w.a_first = (DKV ? u.slot : slots - 1 - u.slot) * kStand;
    w.a_rows = min(kStand, len - w.a_first);
    if (DKV) {
        w.kvh = w.head = p.by_parts.div(u.fast);
        w.part = u.fast - w.kvh * p.parts;
        const int per = p.by_parts.div(p.group + p.parts - 1);
        w.h0 = w.kvh * p.group + min(w.part * per, p.group);
        w.h1 = w.kvh * p.group + min(w.part * per + per, p.group);
    } else {
        w.head = w.h0 = u.fast;
        w.h1 = u.fast + 1;
        w.kvh = p.by_group.div(u.fast);
        w.part = 0;
    }
    int last, unused;
    attn_visible<DKV>(p, u.q.len, u.k.len, w.a_first, w.first, unused);
    attn_visible<DKV>(p, u.q.len, u.k.len, w.a_first + w.a_rows - 1, unused, last);
    w.tiles_per_head = last > w.first ? (last - w.first + kTile - 1) / kTile : 0;
    w.tiles = w.tiles_per_head * (w.h1 - w.h0);
}

template <int HD>
struct Cfg {
    static constexpr int GROUPS = HD == 64 ? 3 : 2, THREADS = (4 * GROUPS + 8) * 32;
    static constexpr int BLOCKS = HD / 64;                                // column blocks of 64 (128 swizzled bytes)
    static constexpr int BLOCK = kTile * 128, TILE = BLOCKS * BLOCK, STAGE = 2 * TILE;
    static constexpr int A_BLOCK = kStand * 128, A_TILE = BLOCKS * A_BLOCK, A_BYTES = 2 * A_TILE;
    static constexpr int UNITS = HD == 64 ? 2 : 1;                        // units whose standing rows are there: what 227 KB hold next to the ring
    static constexpr int STAGES = HD == 64 ? 6 : 4;                       // two more than groups at least, for the loads on their way
    static constexpr int RING = UNITS * A_BYTES, OUT = RING + STAGES * STAGE; // OUT: 2 KB a warp for results on their way out
    static constexpr int ROWS = OUT + 4 * 2048, ROWS_BYTES = GROUPS * 4 * 2 * kTile * 8;
    static constexpr int SLOTS = ROWS + ROWS_BYTES, BARS = SLOTS + kUnitSlots * (int)sizeof(Unit), SMEM = BARS + 448;
    static constexpr int ACC = GROUPS * 2 * kTile;                        // tensor memory: S and dP of each group, then two accumulators
    static_assert(ACC + 2 * HD <= 512 && SMEM <= 227 * 1024 && STAGES >= GROUPS + 2 && BARS % 8 == 0, "");
    static_assert(ROWS_BYTES >= 2 * GROUPS * kStand * 4, "");             // the groups' row sums of two units use the same place
};

template <int HD, bool DKV>
__global__ void __launch_bounds__(Cfg<HD>::THREADS, 1) k_attn_bwd(const __grid_constant__ AttnDev p) {
    using C = Cfg<HD>;
    constexpr int NG = C::GROUPS;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* const full = (uint64_t*)(smem + C::BARS);
    uint64_t *const empty = full + C::STAGES, *const a_full = empty + C::STAGES, *const a_empty = a_full + C::UNITS, *const s_full = a_empty + C::UNITS, *const dp_full = s_full + NG,
                    *const p_full = dp_full + NG, *const ds_full = p_full + NG, *const p_added = ds_full + NG, *const ds_added = p_added + NG, *const acc_done = ds_added + NG, *const acc_free = acc_done + 1, *const sum_full = acc_free + 1, *const sum_empty = sum_full + 2,
                    *const u_full = sum_empty + 2,
                    *const u_empty = u_full + kUnitSlots;
    uint32_t* const tmem_slot = (uint32_t*)(u_empty + kUnitSlots);
    static_assert((2 * C::STAGES + 2 * C::UNITS + 6 * NG + 6 + 2 * kUnitSlots) * 8 + 4 <= 448, "");
    Unit* const slots = (Unit*)(smem + C::SLOTS);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < C::UNITS; ++i) {
            mbar_init(&a_full[i], 1);
            mbar_init(&a_empty[i], NG);  // each group's S and dP are formed
        }
        for (int i = 0; i < NG; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&dp_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&ds_full[i], 128);
            mbar_init(&p_added[i], 1);
            mbar_init(&ds_added[i], 1);
        }
        mbar_init(acc_done, 1);
        mbar_init(acc_free, 4);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sum_full[i], 4 * NG);
            mbar_init(&sum_empty[i], 4);
        }
        for (int i = 0; i < kUnitSlots; ++i) {
            mbar_init(&u_full[i], 1);
            mbar_init(&u_empty[i], NG + 4 * NG + 4);
        }
        fence_mbar_init();
    }
    // The first warp works out the units. Its first one does not need the barriers.
    AttnWalk walk;
    Unit w;
    auto next = [&]() {
        AttnUnit u;
        w.tiles = -1;
        if (next_unit<DKV>(p, walk, u, [](int len) { return (len + kStand - 1) / kStand; })) unit_of<DKV>(p, u, w);
    };
    if (warp == 0) {
        if (lane == 0) {
            prefetch_tmap(&p.tm[0]);
            prefetch_tmap(&p.tm[1]);
            prefetch_tmap(&p.tmA[0]);
            prefetch_tmap(&p.tmA[1]);
        }
        __syncwarp();
        next();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();
    bool ok = true;  // every wait of this warp so far has ended
    // a reader's copy of the index-th unit of the block
    auto take = [&](int index) {
        const int slot = index % kUnitSlots;
        const bool there = __all_sync(0xffffffffu, wait_barrier(&u_full[slot], (uint32_t)(index / kUnitSlots) & 1u, p.status, DEV_ERR_FULL_WAIT));
        w = slots[slot];
        if (!there) w.tiles = -1;
        ok = ok && there;
        __syncwarp();
        if (lane == 0) mbar_arrive(&u_empty[slot]);
        return w.tiles >= 0;
    };

    // 640 threads of 96 registers (64 columns a head), dealt out again: 4 * (48 + 3 * 120 + 72) = 20 * 96 a lane
    if (warp < 4) {
        if (HD == 64) reg_dec<48>();
        if (warp == 0) {
            // ---- units, and by TMA their standing rows, then their tiles
            const uint32_t base = smem_u32(smem), bar = smem_u32(full), a_bar = smem_u32(a_full);
            auto wait = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, wait_barrier(b, parity, p.status, DEV_ERR_EMPTY_WAIT)); };
            int item = 0, st = 0;
            uint32_t round = 0;
            for (int index = 0; ok; ++index) {
                const int slot = index % kUnitSlots;
                if (index >= kUnitSlots) ok = wait(&u_empty[slot], (uint32_t)(index / kUnitSlots - 1) & 1u);
                if (!ok) break;
                if (lane == 0) {
                    slots[slot] = w;
                    mbar_arrive(&u_full[slot]);
                }
                __syncwarp();
                if (w.tiles < 0) break;
                if (w.tiles > 0) {
                    const int ab = item % C::UNITS;
                    if (item >= C::UNITS) ok = wait(&a_empty[ab], (uint32_t)(item / C::UNITS - 1) & 1u);
                    if (!ok) break;
                    mbar_arrive_expect_tx_elect(a_bar + ab * 8, C::A_BYTES);
                    const int a_row = (DKV ? w.k_first : w.q_first) + w.a_first, a_heads = DKV ? p.kv_heads : p.heads;
                    load_head<C::BLOCKS>(&p.tmA[0], base + ab * C::A_BYTES, C::A_BLOCK, a_heads, w.head, a_row, a_bar + ab * 8);
                    load_head<C::BLOCKS>(&p.tmA[1], base + ab * C::A_BYTES + C::A_TILE, C::A_BLOCK, a_heads, w.head, a_row, a_bar + ab * 8);
                    ++item;
                }
                int h = w.h0, t = 0;
                for (int j = 0; j < w.tiles && ok; ++j) {
                    if (round > 0) ok = wait(&empty[st], (round - 1) & 1u);
                    if (!ok) break;
                    const uint32_t b = bar + st * 8, dst = base + C::RING + st * C::STAGE;
                    mbar_arrive_expect_tx_elect(b, C::STAGE);
                    const int row = (DKV ? w.q_first : w.k_first) + w.first + t * kTile;
                    load_head<C::BLOCKS>(&p.tm[0], dst, C::BLOCK, DKV ? p.heads : p.kv_heads, DKV ? h : w.kvh, row, b);
                    load_head<C::BLOCKS>(&p.tm[1], dst + C::TILE, C::BLOCK, DKV ? p.heads : p.kv_heads, DKV ? h : w.kvh, row, b);
                    if (++t == w.tiles_per_head) {
                        t = 0;
                        ++h;
                    }
                    if (++st == C::STAGES) {
                        st = 0;
                        ++round;
                    }
                }
                if (ok) next();
            }
        } else if (warp <= NG) {
            // ---- products of one group
            const int g = warp - 1, before = g == 0 ? NG - 1 : g - 1;
            constexpr uint32_t idesc_s = umma_idesc_bf16(kStand, kTile), idesc_acc = umma_idesc_bf16(kStand, HD) | (1u << 16);  // streamed tile: its K extent in rows
            const uint32_t base = smem_u32(smem), buf = tmem + g * 2 * kTile;
            const uint64_t a_d = umma_desc_k128(base), k_d = umma_desc_k128(base + C::RING), n_d = umma_desc_n128(base + C::RING, C::BLOCK);
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, wait_barrier(bar, parity, p.status, code)); };
            auto product = [&](uint32_t d, int which, int ab, int st) {
                const uint64_t a = a_d + (uint64_t)(uint32_t)((ab * C::A_BYTES + which * C::A_TILE) >> 4), b = k_d + (uint64_t)(uint32_t)((st * C::STAGE + which * C::TILE) >> 4);
#pragma unroll
                for (int i = 0; i < C::BLOCKS; ++i) umma_bf16_x4<2, 2>(d, a + i * (C::A_BLOCK >> 4), b + i * (C::BLOCK >> 4), idesc_s, i > 0);
            };
            auto accumulate = [&](uint32_t d, uint32_t a, int which, int st, bool more) {
                static_assert(kTile == 64, "four products of 16 rows");
                umma_bf16_ts_x4<8, 128>(d, a, n_d + (uint64_t)(uint32_t)((st * C::STAGE + which * C::TILE) >> 4), idesc_acc, more);
            };
            auto need = [&](uint64_t* bar, uint32_t parity, int code) { ok = ok && wait(bar, parity, code); };
            // Two of them, both at once where that is likely: a look at a barrier costs 90 cycles even if it is ready.
        auto need_both = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
            if (!__all_sync(0xffffffffu, mbar_test_wait(a, pa) & mbar_test_wait(b, pb))) {
                need(a, pa, DEV_ERR_ACC_WAIT);
                need(b, pb, DEV_ERR_ACC_WAIT);
            }
        };
        auto there = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test_wait(bar, parity)); };
            // The walk over this group's tiles, which S and dP are at.
            int index = 0, item = -1, seen = -1;  // units taken; units with tiles, less one; the last of those whose standing rows are known to be there
            int t = g, in_head = g, st = g;       // the tile in its unit, in its head; its stage. The first tile of this group is tile g of all.
            uint32_t parity = 0;                  // of the stage
            bool more = true;
            w.tiles = 0;
            auto standing = [&]() {
                if (seen != item) need(&a_full[item % C::UNITS], (uint32_t)(item / C::UNITS) & 1u, DEV_ERR_FULL_WAIT);
                seen = item;
            };
            // To the next tile, not past `units` more units: a later one waits for results that this warp may owe products to. False if that is too
            // far, or there is no more. A unit's standing rows are left behind: every group sees that they were there, also where it has no tile of the unit, since
            // a barrier's parity tells only the next phase from the last one.
            auto find = [&](int units) {
                while (more && t >= w.tiles) {
                    if (units == 0) return false;
                    --units;
                    if (w.tiles > 0) {
                        standing();
                        umma_commit_elect(&a_empty[item % C::UNITS]);
                    }
                    t -= w.tiles;
                    more = ok && take(index++);
                    if (!more) w.tiles = 0;
                    item += w.tiles > 0;
                    in_head = t;
                }
                return more;
            };
            // S or dP of the tile that the walk is at
            auto scores = [&](int which) {
                const int ab = item % C::UNITS;
                if (which == 0) {
                    standing();
                    need(&full[st], parity, DEV_ERR_FULL_WAIT);
                    while (in_head >= w.tiles_per_head) in_head -= w.tiles_per_head;
                    const int valid = (DKV ? w.q_len : w.k_len) - w.first - in_head * kTile;
                    if (ok && valid < kTile) zero_rows(smem + C::RING + st * C::STAGE, C::BLOCK, 2 * C::BLOCKS, valid, kTile);
                    tc_fence_after();
                }
                if (!ok) return;
                product(buf + which * kTile, which, ab, st);
                umma_commit_elect(which ? &dp_full[g] : &s_full[g]);
            };
            bool have = false, early = false;
            for (uint32_t mine = 0;; ++mine) {
                if (!have && more) have = find(INT32_MAX);
                if (!ok || !have) break;
                if (!early) scores(0);
                scores(1);
                const int at = st, unit = item;
                const bool first = t == 0, last = t == w.tiles - 1, follows = g > 0 || mine > 0;
                const uint32_t turns = (g > 0 ? mine : mine - 1) & 1u;  // of the group whose tile is before this one
                t += NG;
                in_head += NG;
                st += NG;
                if (st >= C::STAGES) {
                    st -= C::STAGES;
                    parity ^= 1u;
                }
                // M += P K or dV += P^T dO, behind the tile before; then S of the next tile in P's place while the group is at dS
                if (follows)
                    need_both(&p_full[g], mine & 1u, &p_added[before], turns);
                else
                    need(&p_full[g], mine & 1u, DEV_ERR_ACC_WAIT);
                // the results of the unit before have left the accumulators (behind the tile before, which has seen those of the unit before that leave)
                if (first && unit > 0) need(acc_free, (uint32_t)(unit - 1) & 1u, DEV_ERR_ACC_WAIT);
                if (!ok) break;
                tc_fence_after();
                accumulate(tmem + C::ACC, buf, DKV ? 1 : 0, at, !first);
                umma_commit_elect(&p_added[g]);
                have = find(1);
                // where the next tile is not there yet, dS comes first
                early = have && (seen == item || there(&a_full[item % C::UNITS], (uint32_t)(item / C::UNITS) & 1u)) && there(&full[st], parity);
                if (early) scores(0);
                if (follows)
                    need_both(&ds_full[g], mine & 1u, &ds_added[before], turns);
                else
                    need(&ds_full[g], mine & 1u, DEV_ERR_ACC_WAIT);
                if (!ok) break;
                tc_fence_after();
                accumulate(tmem + C::ACC + HD, buf + kTile, 0, at, !first);
                umma_commit_elect(&ds_added[g]);
                umma_commit_elect(&empty[at]);
                if (last) umma_commit_elect(acc_done);
            }
        }
    } else if (warp < 4 + 4 * NG) {
        // ---- P and dS
        if (HD == 64) reg_inc<120>();
        const int group = (warp >> 2) - 1, r = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, buf = tmem + lanes + group * 2 * kTile;
        // -lse and -D of streamed queries, twice. Each warp has its own: a barrier of the group's four would be one without a limit, or cost more than the loads
        // (1 x 8 192, 28 / 4 heads of 128, whole backward pass: one copy behind a barrier in shared memory takes 4% longer).
        float* const stats = (float*)(smem + C::ROWS) + (warp - 4) * 4 * kTile;
        // A wait that ran out lets the warp go on without waiting, since the others wait for it at their barriers.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait_barrier(bar, parity, p.status, DEV_ERR_ACC_WAIT));
            tc_fence_after();
        };
        int item = 0, turn = 0;  // units with tiles so far; tiles of all units before, modulo the groups
        uint32_t mine = 0;       // tiles of this group so far
        const F2 scale2 = f2(p.scale_log2, p.scale_log2);
        for (int index = 0; take(index); ++index) {
            const bool live = r < w.a_rows;
            const int row = w.a_first + r, grow = (DKV ? w.k_first : w.q_first) + row;  // row of the sequence, of the buffers
            int lo = 0, hi = 0;
            if (live) attn_visible<DKV>(p, w.q_len, w.k_len, row, lo, hi);
            float nl = 0.f, nd = 0.f, sum = 0.f;  // -lse, -D
            if (!DKV && live) {
                const float l = p.lse[(int64_t)w.head * p.rows_q + grow];
                nl = l == -INFINITY ? 0.f : -l * kLog2e;
                nd = -__ldcg(p.d + (int64_t)w.head * p.rows_q + grow);
            }
            int t = group - turn;  // this group's first tile of the unit
            if (t < 0) t += NG;
            int h = w.h0, in_head = t;
            auto settle = [&]() {
                while (in_head >= w.tiles_per_head && h < w.h1) {
                    in_head -= w.tiles_per_head;
                    ++h;
                }
            };
            // lse and D of a tile's queries, two each
            float l_ahead[2] = {0.f, 0.f}, d_ahead[2] = {0.f, 0.f};
            auto fetch = [&]() {
                const int col = w.first + in_head * kTile + lane;
                const int64_t at = (int64_t)h * p.rows_q + w.q_first + col;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const bool there = h < w.h1 && col + 32 * i < w.q_len;
                    l_ahead[i] = there ? __ldg(p.lse + at + 32 * i) : -INFINITY;
                    d_ahead[i] = there ? __ldcg(p.d + at + 32 * i) : 0.f;
                }
            };
            if (w.tiles > 0) settle();
            if (DKV && t < w.tiles) fetch();
            for (; t < w.tiles; t += NG, ++mine) {
                const uint32_t ph = mine & 1u;
                const int first = w.first + in_head * kTile, c_lo = lo - first, c_hi = hi - first;  // visible columns
                const bool whole = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= kTile);
                float* const q_stats = stats + ph * 2 * kTile;
                in_head += NG;
                settle();
                if (DKV) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        q_stats[lane + 32 * i] = l_ahead[i] == -INFINITY ? 0.f : -l_ahead[i] * kLog2e;
                        q_stats[kTile + lane + 32 * i] = -d_ahead[i];
                    }
                    fetch();
                    __syncwarp();
                }
                wait(&s_full[group], ph);
                F2 pr[kTile / 2];
                uint64_t seen = 0;
                if (!whole) seen = bits_between(c_lo, c_hi);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t s[2][16], v[16];
                    tmem_ld16(buf + half * 32, s[0]);
                    tmem_ld16(buf + half * 32 + 16, s[1]);
                    tc_wait_ld();
                    if (!whole)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (!((uint32_t)(seen >> (half * 32)) & 1u << i)) s[i >> 4][i & 15] = 0xff800000u;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 l4 = make_float4(nl, nl, nl, nl);
                        if constexpr (DKV) l4 = *(const float4*)(q_stats + half * 32 + i);
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const int k = i + e;
                            float x, y;
                            split2(fma2(f2(__uint_as_float(s[k >> 4][k & 15]), __uint_as_float(s[k >> 4][(k & 15) + 1])), scale2, e ? f2(l4.z, l4.w) : f2(l4.x, l4.y)), x, y);
                            x = exp2_fast(x);
                            y = exp2_fast(y);
                            pr[(half * 32 + k) >> 1] = f2(x, y);
                            v[k >> 1] = pack2(x, y);
                        }
                    }
                    tmem_st16(buf + half * 16, v);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[group]);
                wait(&dp_full[group], ph);
                F2 part = 0ull;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t s[2][16], v[16];
                    tmem_ld16(buf + kTile + half * 32, s[0]);
                    tmem_ld16(buf + kTile + half * 32 + 16, s[1]);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 d4 = make_float4(nd, nd, nd, nd);
                        if constexpr (DKV) d4 = *(const float4*)(q_stats + kTile + half * 32 + i);
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const int k = i + e;
                            const F2 ds = mul2(pr[(half * 32 + k) >> 1],
                                               add2(f2(__uint_as_float(s[k >> 4][k & 15]), __uint_as_float(s[k >> 4][(k & 15) + 1])), e ? f2(d4.z, d4.w) : f2(d4.x, d4.y)));
                            if constexpr (!DKV) part = add2(part, ds);
                            float x, y;
                            split2(ds, x, y);
                            v[k >> 1] = pack2(x, y);
                        }
                    }
                    tmem_st16(buf + kTile + half * 16, v);
                }
                if constexpr (!DKV) {
                    float x, y;
                    split2(part, x, y);
                    sum += x + y;
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&ds_full[group]);
            }
            turn = (turn + w.tiles) % NG;
            if (!DKV && w.tiles > 0) {
                const int at = item & 1;
                if (item >= 2) wait(&sum_empty[at], (uint32_t)(item / 2 - 1) & 1u);
                ((float*)(smem + C::ROWS))[(at * NG + group) * kStand + r] = sum;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sum_full[at]);
            }
            item += w.tiles > 0;
        }
    } else {
        // ---- results
        if (HD == 64) reg_dec<72>();
        const int r = tid & 127, warp_row = (warp & 3) * 32;
        const uint32_t lanes = (uint32_t)warp_row << 16;
        uint8_t* const out = smem + C::OUT + (warp & 3) * 2048;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait_barrier(bar, parity, p.status, DEV_ERR_ACC_WAIT));
            tc_fence_after();
        };
        int item = 0;
        for (int index = 0; take(index); ++index) {
            const bool live = r < w.a_rows;
            const int rows = w.a_rows - warp_row, grow = (DKV ? w.k_first : w.q_first) + w.a_first + r, grow0 = grow - lane;  // rows of the buffers
            if (w.tiles == 0) {  // nothing is seen: zeros
                if (live)
                    for (int k = 0; k < (DKV ? 2 : 1) * p.hd / 8; ++k) {
                        const bool second = k >= p.hd / 8;
                        const int c = (second ? k - p.hd / 8 : k) * 8;
                        if (DKV && p.partial) {
                            float* const to = p.partial + ((((int64_t)(second ? p.parts : 0) + w.part) * p.rows_k + grow) * p.kv_heads + w.kvh) * p.hd + c;
                            *(uint4*)to = *(uint4*)(to + 4) = make_uint4(0u, 0u, 0u, 0u);
                        } else {
                            *(uint4*)((second ? p.out1 + grow * p.out1_stride : p.out0 + grow * p.out0_stride) + (int64_t)w.head * p.hd + c) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                continue;
            }
            float sum = 0.f, d = 0.f;
            float* const d_at = p.d + (int64_t)w.head * p.rows_q + grow;
            if (!DKV && live) d = __ldcg(d_at);
            wait(acc_done, (uint32_t)item & 1u);
            if constexpr (!DKV) {
                const int at = item & 1;
                wait(&sum_full[at], (uint32_t)(item / 2) & 1u);
#pragma unroll
                for (int g = 0; g < NG; ++g) sum += ((const float*)(smem + C::ROWS))[(at * NG + g) * kStand + r];
                __syncwarp();
                if (lane == 0) mbar_arrive(&sum_empty[at]);
                if (live) *d_at = d + sum;
            }
            ++item;
            // 64 bytes of a row at a time, 32 columns or 16 of an fp32 sum
            auto store = [&](auto wide) {
                constexpr int COLS = wide.value ? 16 : 32, PER = HD / COLS, PIECES = (DKV ? 2 : 1) * PER;
#pragma unroll 1
                for (int k = 0; k < PIECES; ++k) {
                    const bool second = DKV && k >= PER;  // dV
                    const int c = (k - (second ? PER : 0)) * COLS;
                    const float f = second ? 1.f : p.scale;
                    float v[COLS];
                    uint32_t a[COLS / 16][16];
#pragma unroll
                    for (int i = 0; i < COLS / 16; ++i) tmem_ld16(tmem + lanes + C::ACC + (second ? 0 : HD) + c + 16 * i, a[i]);
                    if constexpr (!DKV) {
                        uint32_t m[COLS / 16][16];
#pragma unroll
                        for (int i = 0; i < COLS / 16; ++i) tmem_ld16(tmem + lanes + C::ACC + c + 16 * i, m[i]);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < COLS; ++i) v[i] = f * fmaf(-sum, __uint_as_float(m[i >> 4][i & 15]), __uint_as_float(a[i >> 4][i & 15]));
                    } else {
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < COLS; ++i) v[i] = f * __uint_as_float(a[i >> 4][i & 15]);
                    }
                    if (k == PIECES - 1) {  // the last look at the accumulators
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_free);
                    }
                    uint4 x[4];
                    char* to;
                    int64_t stride;
                    if constexpr (wide.value) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
                        stride = (int64_t)p.kv_heads * p.hd * 4;
                        to = (char*)p.partial + (((int64_t)(second ? p.parts : 0) + w.part) * p.rows_k + grow0) * stride + ((int64_t)w.kvh * p.hd + c) * 4;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = make_uint4(pack2(v[8 * i], v[8 * i + 1]), pack2(v[8 * i + 2], v[8 * i + 3]), pack2(v[8 * i + 4], v[8 * i + 5]), pack2(v[8 * i + 6], v[8 * i + 7]));
                        stride = (second ? p.out1_stride : p.out0_stride) * 2;
                        to = (char*)(second ? p.out1 : p.out0) + grow0 * stride + ((int64_t)w.head * p.hd + c) * 2;
                    }
                    store_rows(out, x, to, stride, rows, (p.hd - c) * (wide.value ? 4 : 2) / 16);
                }
            };
            if (DKV && p.partial)
                store(std::true_type());
            else
                store(std::false_type());
        }
    }
    tc_fence_before();
    if (__syncthreads_or(!ok)) let_land();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

// D'[h][row] = sum of dO o O over the head: L = HD / 8 lanes a row, neighbouring rows in neighbouring lanes, four rows a lane in flight
template <int L>
__global__ void __launch_bounds__(256) k_attn_dot(const bf16* __restrict__ d_out, const bf16* __restrict__ out, int64_t stride, const int* cu_q, int n_seqs, int64_t rows, int heads,
                                                  int hd, float* __restrict__ d) {
    constexpr int ROWS = 256 / L;
    pdl_launch_dependents();
    const int64_t row0 = (int64_t)blockIdx.x * (4 * ROWS) + threadIdx.x / L;
    const int h = blockIdx.y, c = threadIdx.x % L * 8;
    const int64_t begin = cu_q[0], end = min((int64_t)cu_q[n_seqs], rows);
    uint4 x[4], y[4];  // of rows in front of the first sequence and behind the last as well, which are not waited for to be told apart
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + i * ROWS;
        x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows && c < hd) {
            x[i] = __ldg((const uint4*)(d_out + row * stride + (int64_t)h * hd + c));
            y[i] = __ldg((const uint4*)(out + row * stride + (int64_t)h * hd + c));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = row0 + i * ROWS;
        const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a = fmaf(bf16_lo(xs[k]), bf16_lo(ys[k]), a);
            a = fmaf(bf16_hi(xs[k]), bf16_hi(ys[k]), a);
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (row >= begin && row < end && c == 0) d[(int64_t)h * rows + row] = a;
    }
}

// dK and dV from the parts of the query heads, added in their order; kJoinRows rows a block
constexpr int kJoinRows = 8;
__global__ void __launch_bounds__(256) k_attn_join(const float* __restrict__ partial, int parts, const int* cu_k, int n_seqs, int64_t rows, int kv_heads, int hd, bf16* dk,
                                                   int64_t dk_stride, bf16* dv, int64_t dv_stride) {
    const int per_row = kv_heads * hd / 4;
    const int64_t plane = rows * kv_heads * hd;
    const float* src = partial + (int64_t)blockIdx.y * parts * plane;
    const int begin = cu_k[0], end = cu_k[n_seqs];
    pdl_wait();
    for (int i = threadIdx.x; i < kJoinRows * per_row; i += 256) {
        const int r = i / per_row, c = (i - r * per_row) * 4;
        const int64_t row = (int64_t)blockIdx.x * kJoinRows + r;
        if (row >= rows || row < begin || row >= end) continue;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int q = 0; q < parts; ++q) {
            const float4 v = __ldcg((const float4*)(src + q * plane + row * kv_heads * hd + c));
            a.x += v.x;
            a.y += v.y;
            a.z += v.z;
            a.w += v.w;
        }
        bf16* dst = blockIdx.y ? dv + row * dv_stride : dk + row * dk_stride;
        *(uint2*)(dst + c) = make_uint2(pack2(a.x, a.y), pack2(a.z, a.w));
    }
}

template <int HD, bool DKV>
int run(AttnDev& p, int64_t units, int num_sms, cudaStream_t s, bool pdl) {
    using C = Cfg<HD>;
    const cudaError_t e = allow_shared<k_attn_bwd<HD, DKV>>(C::SMEM);
    if (e != cudaSuccess) return (int)e;
    const unsigned grid = set_units(p, units, num_sms);
    return (int)launch_k(k_attn_bwd<HD, DKV>, dim3(grid), dim3(C::THREADS), (size_t)C::SMEM, s, pdl, p);
}

// Parts of the query heads of a kv head for dK, dV. One block adds all of them up where there are one and a half units of work for each of the
// 148 SMs, as the packed rows let expect (one, if sequences are so short that the join costs as much as the last units); else the heads are dealt to as many units as that takes, and their sums are joined through the workspace.
// All heads together against this, us, whole call: 1 x 4 096, 14 / 2 heads of 64 296 against 134; 8 ragged x 2 048, 12 / 2 of 128 228 against 175.
// One unit an SM against one and a half: 1 x 4 096, 14 / 2 of 64 168 against 137; 20 ragged x 1 000 of them 114 against 111, 24 x 700 87 against 91,
// 32 x 512 73 against 79. Parts of single heads against this: 8 x 4 096, 14 / 2 of 64 986 against 852; 1 x 8 192, 28 / 4 of 128 1 415 against 1 363.
int parts_of(const AttnCall& c) {
    const int G = c.heads / c.kv_heads;
    const int64_t most = std::min((int64_t)((c.max_k + kStand - 1) / kStand) * c.n_seqs, kMostUnits) * c.kv_heads, expected = (c.rows_k / kStand + c.n_seqs / 2) * c.kv_heads, units = std::max<int64_t>(std::min(most, expected), 1);
    const int64_t enough = c.max_k > 768 ? 148 * 3 / 2 : 148;
    int parts = 1;
    while (parts < G && units * parts < enough) ++parts;
    const int per = (G + parts - 1) / parts;
    return (G + per - 1) / per;
}
int64_t d_bytes(const AttnCall& c) { return ((int64_t)c.heads * c.rows_q * 4 + 255) / 256 * 256; }

}  // namespace

int64_t attention_workspace_bytes(const AttnCall& c) {
    const int parts = parts_of(c);
    return d_bytes(c) + (parts > 1 ? 2 * parts * c.rows_k * c.kv_heads * c.hd * 4 : 0);
}

bool attention_backward_fits(const AttnCall& c) {
    return blocks_of_rows(c, c.max_q, c.rows_q) * c.heads < kMostUnits && blocks_of_rows(c, c.max_k, c.rows_k) * c.kv_heads * parts_of(c) < kMostUnits;
}

int launch_attention_train_backward(const AttnCall& c, int num_sms, cudaStream_t s) {
    const bool queries = c.max_q > 0 && c.rows_q > 0, keys = c.max_k > 0 && c.rows_k > 0;
    if (c.n_seqs == 0 || (!queries && !keys)) return 0;
    float* const d = (float*)c.workspace;
    AttnDev p = attn_dev(c);
    p.d = d;
    p.chunk_slots = c.chunk > 0 ? std::max(c.chunk / kStand, 1) : 0;
    // without keys or without queries: any valid map stands in, none of its rows is read
    CUtensorMap q64, g64, k64, v64, q128, g128, k128, v128;
    const AttnCall& a = c;
    if (queries && (!map_heads(&q64, a.q, a.rows_q, a.q_stride, a.heads, a.hd, kTile) || !map_heads(&g64, a.d_out, a.rows_q, a.out_stride, a.heads, a.hd, kTile) ||
                    !map_heads(&q128, a.q, a.rows_q, a.q_stride, a.heads, a.hd, kStand) || !map_heads(&g128, a.d_out, a.rows_q, a.out_stride, a.heads, a.hd, kStand)))
        return -1000;
    if (keys && (!map_heads(&k64, a.k, a.rows_k, a.k_stride, a.kv_heads, a.hd, kTile) || !map_heads(&v64, a.v, a.rows_k, a.v_stride, a.kv_heads, a.hd, kTile) ||
                 !map_heads(&k128, a.k, a.rows_k, a.k_stride, a.kv_heads, a.hd, kStand) || !map_heads(&v128, a.v, a.rows_k, a.v_stride, a.kv_heads, a.hd, kStand)))
        return -1000;
    if (!keys) k64 = v64 = q64;
    if (!queries) q64 = g64 = k64;
    int rc = 0;
    if (queries) {
        const int lanes = c.hd <= 64 ? 8 : 16;
        const dim3 grid((unsigned)((c.rows_q + 1024 / lanes - 1) / (1024 / lanes)), (unsigned)c.heads);
        rc = lanes == 8 ? (int)launch_k(k_attn_dot<8>, grid, dim3(256), 0, s, false, c.d_out, (const bf16*)c.out, c.out_stride, c.cu_q, c.n_seqs, c.rows_q, c.heads, c.hd, d)
                        : (int)launch_k(k_attn_dot<16>, grid, dim3(256), 0, s, false, c.d_out, (const bf16*)c.out, c.out_stride, c.cu_q, c.n_seqs, c.rows_q, c.heads, c.hd, d);
        if (rc) return rc;
        const int64_t units = blocks_of_rows(c, c.max_q, c.rows_q) * c.heads;
        p.by_fast = FastDiv::of(c.heads);
        p.tm[0] = k64;
        p.tm[1] = v64;
        p.tmA[0] = q128;
        p.tmA[1] = g128;
        p.out0 = c.dq;
        p.out0_stride = c.q_stride;
        rc = c.hd <= 64 ? run<64, false>(p, units, num_sms, s, true) : run<128, false>(p, units, num_sms, s, true);
        if (rc) return rc;
    }
    if (keys) {
        p.parts = parts_of(c);
        p.partial = p.parts > 1 ? (float*)((char*)c.workspace + d_bytes(c)) : nullptr;
        const int64_t units = blocks_of_rows(c, c.max_k, c.rows_k) * c.kv_heads * p.parts;
        p.by_fast = FastDiv::of(c.kv_heads * p.parts);
        p.by_parts = FastDiv::of(p.parts);
        p.tm[0] = q64;
        p.tm[1] = g64;
        p.tmA[0] = k128;
        p.tmA[1] = v128;
        p.out0 = c.dk;
        p.out0_stride = c.k_stride;
        p.out1 = c.dv;
        p.out1_stride = c.v_stride;
        rc = c.hd <= 64 ? run<64, true>(p, units, num_sms, s, queries) : run<128, true>(p, units, num_sms, s, queries);
        if (rc) return rc;
        if (p.partial) {
            rc = (int)launch_k(k_attn_join, dim3((unsigned)((c.rows_k + kJoinRows - 1) / kJoinRows), 2), dim3(256), 0, s, true, (const float*)p.partial, p.parts, c.cu_k, c.n_seqs,
                               c.rows_k, c.kv_heads, c.hd, c.dk, c.k_stride, c.dv, c.v_stride);
        }
    }
    return rc;
}

}  // namespace tffn
