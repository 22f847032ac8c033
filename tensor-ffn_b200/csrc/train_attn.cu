// Forward pass of the attention of packed training sequences on the tensor cores (inference/src/model/qwen.cu:349-412 materialises the scores):
//   S = scale Q K^T inside the mask,   O = softmax(S) V,   lse = log of the softmax's denominators
//
// A persistent block of three (64 columns a head) or two (128) groups of four warps streams tiles of 64 keys and values past units of 128 queries of
// one head (thread = query). With few units the groups take turns at the tiles of one unit, each with a maximum, a sum and an O of its own that
// are joined at its end, so that a unit is done sooner and uneven lengths even out; with many, each group has a unit to itself, mostly
// heads of the same queries, which share what is fetched. S = Q K^T and O += P V are tcgen05 products. One warp works out the units and fills the
// rings by TMA, one per group issues its products. S has its columns to itself and P others, so the next S is formed as soon as a group has S
// in registers, and a group's exponentials follow each other without waiting for the tensor cores. The next unit's queries and scores are on their
// way while results are stored. S, sums and O are fp32; P enters its product as bf16 (half a step, up to 2^-8 of each term, as inputs and results
// have). A row's reference maximum moves only when it would be passed by more than 2^8, so O is rarely rescaled.
//
// What bounds it: 64 columns a head: the exponentials (8 192 a tile at 16 a cycle), a quarter of which therefore run as polynomials on the FMA
// pipe (8 x 4 096, 14 / 2 heads: 325 us, 0.74 PFLOP/s); 128: the products (640 cycles a tile; 1 x 8 192, 28 / 4 heads: 458 us, 1.05 PFLOP/s in a row of
// calls, under the power limit); short sequences: the chain from a unit's queries to its results (32 ragged x 512, 14 / 2 heads of 64: 30 us, 0.17).
#include "train_attn.cuh"
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace tffn {

namespace {

constexpr int kTile = 64;

// up to NG units of one kv head of a sequence, or one unit that the groups share, and the tiles of keys that any of them sees
template <int NG>
struct Units {
    int q_first, k_first, q_len, k_len, kvh;
    int first, tiles;  // tiles = -1: no more work
    int n;
    int a_first[NG], a_rows[NG], head[NG];
};

// the units of one step of a block's walk
template <int NG>
__device__ __forceinline__ void units_of(const AttnDev& p, const AttnUnit& u, Units<NG>& w) {
    w.q_first = u.q.first;
    w.k_first = u.k.first;
    w.q_len = u.q.len;
    w.k_len = u.k.len;
    w.kvh = u.fast;
    const int blocks = (u.q.len + kStand - 1) / kStand, first_unit = u.slot * p.parts;
    w.n = min(p.parts, blocks * p.group - first_unit);
    int last = 0;
    w.first = INT32_MAX;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        w.a_first[g] = w.a_rows[g] = w.head[g] = 0;
        if (g < w.n) {
            const int unit = first_unit + g, block = p.by_group.div(unit);
            w.head[g] = u.fast * p.group + unit - block * p.group;
            w.a_first[g] = (blocks - 1 - block) * kStand;  // late queries see most keys: first
            w.a_rows[g] = min(kStand, u.q.len - w.a_first[g]);
            int lo, hi, unused;
            attn_visible<false>(p, u.q.len, u.k.len, w.a_first[g], lo, unused);
            attn_visible<false>(p, u.q.len, u.k.len, w.a_first[g] + w.a_rows[g] - 1, unused, hi);
            if (hi > lo) {
                w.first = min(w.first, lo);
                last = max(last, hi);
            }
        }
    }
    w.tiles = last > 0 ? (last - w.first + kTile - 1) / kTile : 0;
}

template <int HD>
struct Cfg {
    static constexpr int GROUPS = HD == 64 ? 3 : 2, THREADS = (4 * GROUPS + 4) * 32;
    static constexpr int BLOCKS = HD / 64, BLOCK = kTile * 128, TILE = BLOCKS * BLOCK;  // column blocks of 64 (128 swizzled bytes)
    static constexpr int Q_BLOCK = kStand * 128, Q_TILE = BLOCKS * Q_BLOCK;
    // Queries of each group, or of the unit that they share; then the stages of the ring, K and V. Groups that share a unit have a part of the ring
    // each: a barrier's parity tells only the next phase from the last one, so whoever waits for a stage has to be the one that saw its last phase.
    static constexpr int OWN_STAGES = 4, PART = HD == 64 ? 3 : 2, STAGE = 2 * TILE;
    static constexpr int own_bytes = GROUPS * Q_TILE + OWN_STAGES * STAGE, shared_bytes = Q_TILE + GROUPS * PART * STAGE;
    static constexpr int OUT = own_bytes > shared_bytes ? own_bytes : shared_bytes;     // 2 KB a warp for its results on their way out
    static constexpr int STATS = OUT + GROUPS * 4 * 2048;
    static constexpr int SLOTS = STATS + GROUPS * kStand * 8, BARS = SLOTS + kUnitSlots * (int)sizeof(Units<GROUPS>), SMEM = BARS + 640;
    static_assert(BARS % 8 == 0, "");
    // tensor memory: S of each group, P of each group, O of each group
    static constexpr int P = GROUPS * kTile, ACC = P + GROUPS * kTile / 2;
    static_assert(ACC + GROUPS * HD <= 512 && SMEM <= 227 * 1024, "");
};

template <int HD>
__global__ void __launch_bounds__(Cfg<HD>::THREADS, 1) k_attn_fwd(const __grid_constant__ AttnDev p) {
    using C = Cfg<HD>;
    constexpr int NG = C::GROUPS, MOST = NG * C::PART;
    extern __shared__ __align__(1024) uint8_t smem[];
    const bool own = p.parts > 1;  // each group has a unit of its own
    const int part = own ? C::OWN_STAGES : C::PART, ring_at = (own ? NG : 1) * C::Q_TILE;
    uint64_t* const k_full = (uint64_t*)(smem + C::BARS);
    uint64_t *const k_empty = k_full + MOST, *const v_full = k_empty + MOST, *const v_empty = v_full + MOST, *const q_full = v_empty + MOST, *const q_empty = q_full + NG,
                    *const s_full = q_empty + NG, *const s_free = s_full + NG, *const p_full = s_free + NG, *const o_full = p_full + NG, *const o_free = o_full + NG,
                    *const joined = o_free + NG, *const u_full = joined + 2, *const u_empty = u_full + kUnitSlots;
    uint32_t* const tmem_slot = (uint32_t*)(u_empty + kUnitSlots);
    Units<NG>* const slots = (Units<NG>*)(smem + C::SLOTS);
    static_assert((4 * MOST + 7 * NG + 2 + 2 * kUnitSlots) * 8 + 4 <= 640 && C::OWN_STAGES <= MOST, "");
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < MOST; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], own ? NG : 1);
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], own ? NG : 1);
        }
        for (int i = 0; i < NG; ++i) {
            mbar_init(&q_full[i], 1);
            mbar_init(&q_empty[i], own ? 1 : NG);
            mbar_init(&s_full[i], 1);
            mbar_init(&s_free[i], 128);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_free[i], 128);
        }
        for (int i = 0; i < 2; ++i) mbar_init(&joined[i], 4 * NG);
        for (int i = 0; i < kUnitSlots; ++i) {
            mbar_init(&u_full[i], 1);
            mbar_init(&u_empty[i], NG + 4 * NG);
        }
        fence_mbar_init();
    }
    // The first warp works out the units. Its first one does not need the barriers.
    AttnWalk walk;
    Units<NG> w;
    auto next_units = [&]() {
        AttnUnit u;
        w.tiles = -1;
        if (next_unit<false>(p, walk, u, [&](int len) { return p.by_parts.div((len + kStand - 1) / kStand * p.group + p.parts - 1); })) units_of<NG>(p, u, w);
    };
    if (warp == 0) {
        if (lane == 0) {
            prefetch_tmap(&p.tm[0]);
            prefetch_tmap(&p.tm[1]);
            prefetch_tmap(&p.tmA[0]);
        }
        __syncwarp();
        next_units();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // a place in a ring, or in a group's part of it
    struct Place {
        int stage = 0;
        uint32_t parity = 0;
        __device__ __forceinline__ void step(int part) {
            if (++stage == part) {
                stage = 0;
                parity ^= 1u;
            }
        }
    };
    bool ok = true;  // every wait of this warp so far has ended
    // a reader's copy of the index-th units of the block; false if there are no more
    auto take = [&](int index) {
        const int slot = index % kUnitSlots;
        const bool there = __all_sync(0xffffffffu, wait_barrier(&u_full[slot], (uint32_t)(index / kUnitSlots) & 1u, p.status, DEV_ERR_FULL_WAIT));
        ok = ok && there;
        w = slots[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&u_empty[slot]);
        return there && w.tiles >= 0;
    };

    if (warp == 0) {
        // ---- units, and by TMA their queries, then keys and values tile by tile
        const uint32_t base = smem_u32(smem);
        auto wait = [&](uint64_t* b, uint32_t parity) { return __all_sync(0xffffffffu, wait_barrier(b, parity, p.status, DEV_ERR_EMPTY_WAIT)); };
        int begun[NG] = {0};
        Place fill[NG];
        uint32_t first_round = (1u << NG) - 1u;  // of each part of the ring
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
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (ok && w.tiles > 0 && g < w.n) {
                    if (begun[g] > 0) ok = wait(&q_empty[g], (uint32_t)(begun[g] - 1) & 1u);
                    if (ok) {
                        mbar_arrive_expect_tx_elect(smem_u32(&q_full[g]), C::Q_TILE);
                        load_head<C::BLOCKS>(&p.tmA[0], base + g * C::Q_TILE, C::Q_BLOCK, p.heads, w.head[g], w.q_first + w.a_first[g], smem_u32(&q_full[g]));
                    }
                    ++begun[g];
                }
            for (int t = 0; t < w.tiles && ok; ++t) {
                const int row = w.k_first + w.first + t * kTile, to = own ? 0 : t % NG;
                Place at = fill[0];
#pragma unroll
                for (int i = 1; i < NG; ++i)
                    if (i == to) at = fill[i];
                const int st = to * (own ? 0 : C::PART) + at.stage;
                const bool fresh = first_round >> to & 1u;
                if (!fresh) ok = wait(&k_empty[st], at.parity ^ 1u);
                if (!ok) break;
                mbar_arrive_expect_tx_elect(smem_u32(&k_full[st]), C::TILE);
                load_head<C::BLOCKS>(&p.tm[0], base + ring_at + st * C::STAGE, C::BLOCK, p.kv_heads, w.kvh, row, smem_u32(&k_full[st]));
                if (!fresh) ok = wait(&v_empty[st], at.parity ^ 1u);
                if (!ok) break;
                mbar_arrive_expect_tx_elect(smem_u32(&v_full[st]), C::TILE);
                load_head<C::BLOCKS>(&p.tm[1], base + ring_at + st * C::STAGE + C::TILE, C::BLOCK, p.kv_heads, w.kvh, row, smem_u32(&v_full[st]));
                at.step(part);
                if (at.stage == 0) first_round &= ~(1u << to);
#pragma unroll
                for (int i = 0; i < NG; ++i)
                    if (i == to) fill[i] = at;
            }
            if (ok) next_units();
        }
    } else if (warp <= NG) {
        // ---- products of one group
        const int g = warp - 1, qb = own ? g : 0, step = own ? 1 : NG, begin = own ? 0 : g;
        constexpr uint32_t idesc_s = umma_idesc_bf16(kStand, kTile), idesc_o = umma_idesc_bf16(kStand, HD) | (1u << 16);  // V: its K extent in rows
        const uint32_t base = smem_u32(smem), s_at = tmem + g * kTile, p_at = tmem + C::P + g * (kTile / 2), o_at = tmem + C::ACC + g * HD;
        const int ring0 = own ? 0 : g * C::PART;  // this group's part
        uint8_t* const ring = smem + ring_at + ring0 * C::STAGE;
        uint64_t *const kf = k_full + ring0, *const ke = k_empty + ring0, *const vf = v_full + ring0, *const ve = v_empty + ring0;
        const uint64_t q_d = umma_desc_k128(base + qb * C::Q_TILE), k_d = umma_desc_k128(smem_u32(ring)), v_d = umma_desc_n128(smem_u32(ring) + C::TILE, C::BLOCK);
        auto wait = [&](uint64_t* bar, uint32_t parity, int code) { ok = ok && __all_sync(0xffffffffu, wait_barrier(bar, parity, p.status, code)); };
        // two at once: a barrier that is ready costs 90 cycles to look at
        auto wait_both = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
            if (!__all_sync(0xffffffffu, mbar_test_wait(a, pa) & mbar_test_wait(b, pb))) {
                wait(a, pa, DEV_ERR_FULL_WAIT);
                wait(b, pb, DEV_ERR_ACC_WAIT);
            }
        };
        auto there = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test_wait(bar, parity)); };
        Place ks, vs;
        auto scores = [&](bool last) {
            tc_fence_after();
            const uint64_t b = k_d + (uint64_t)(uint32_t)((ks.stage * C::STAGE) >> 4);
#pragma unroll
            for (int i = 0; i < C::BLOCKS; ++i) umma_bf16_x4<2, 2>(s_at, q_d + i * (C::Q_BLOCK >> 4), b + i * (C::BLOCK >> 4), idesc_s, i > 0);
            umma_commit_elect(&s_full[g]);
            umma_commit_elect(&ke[ks.stage]);
            if (last) umma_commit_elect(&q_empty[qb]);
            ks.step(part);
        };
        uint32_t turns = 0, units = 0, results = 0;  // tiles of this group so far; units whose queries have come; units with a result of this group
        bool ahead = false;                          // S of the unit's first tile has been issued
        for (int index = 0; ok && take(index); ++index) {
            const int tiles = w.tiles;
            if (own && g >= w.n) {  // no unit for this group: it passes the tiles on
                for (int t = 0; t < tiles && ok; ++t) {
                    wait(&kf[ks.stage], ks.parity, DEV_ERR_FULL_WAIT);
                    if (lane == 0) mbar_arrive(&ke[ks.stage]);
                    ks.step(part);
                    wait(&vf[vs.stage], vs.parity, DEV_ERR_FULL_WAIT);
                    if (lane == 0) mbar_arrive(&ve[vs.stage]);
                    vs.step(part);
                }
                continue;
            }
            const int last_valid = w.k_len - w.first;
            if (begin < tiles && !ahead) {
                wait(&q_full[qb], units & 1u, DEV_ERR_FULL_WAIT);
                wait(&kf[ks.stage], ks.parity, DEV_ERR_FULL_WAIT);
                if (ok) scores(begin + step >= tiles);
            }
            ahead = false;
            if (tiles > 0 && begin >= tiles) {  // fewer tiles than groups: the shared queries are let go all the same, once they are there
                wait(&q_full[qb], units & 1u, DEV_ERR_FULL_WAIT);
                if (ok && lane == 0) mbar_arrive(&q_empty[qb]);
            }
            units += tiles > 0;
            for (int t = begin; t < tiles && ok; t += step, ++turns) {
                // S of the next tile, as soon as the group has this one in registers; of the next unit's first if that is there already
                if (t + step < tiles) {
                    wait_both(&kf[ks.stage], ks.parity, &s_free[g], turns & 1u);
                    if (ok) scores(t + 2 * step >= tiles);
                } else {
                    const int after = index + 1, at = after % kUnitSlots;
                    if (there(&u_full[at], (uint32_t)(after / kUnitSlots) & 1u)) {
                        const int more = slots[at].tiles;
                        if (begin < more && (!own || g < slots[at].n) && there(&q_full[qb], units & 1u) && there(&kf[ks.stage], ks.parity)) {
                            wait(&s_free[g], turns & 1u, DEV_ERR_ACC_WAIT);
                            if (ok) scores(begin + step >= more);
                            ahead = true;
                        }
                    }
                }
                wait(&vf[vs.stage], vs.parity, DEV_ERR_FULL_WAIT);
                const int valid = last_valid - t * kTile;
                if (ok && valid < kTile) zero_rows(ring + vs.stage * C::STAGE + C::TILE, C::BLOCK, C::BLOCKS, valid, kTile);
                if (t == begin && results > 0) wait(&o_free[g], (results - 1) & 1u, DEV_ERR_ACC_WAIT);
                wait(&p_full[g], turns & 1u, DEV_ERR_ACC_WAIT);
                if (!ok) break;
                tc_fence_after();
                umma_bf16_ts_x4<8, 128>(o_at, p_at, v_d + (uint64_t)(uint32_t)((vs.stage * C::STAGE) >> 4), idesc_o, t > begin);
                umma_commit_elect(&o_full[g]);
                umma_commit_elect(&ve[vs.stage]);
                vs.step(part);
            }
            results += begin < tiles;
        }
    } else if (warp >= 4) {
        // ---- softmax
        const int g = (warp >> 2) - 1, r = tid & 127, step = own ? 1 : NG, begin = own ? 0 : g;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_at = tmem + g * kTile, p_at = tmem + C::P + g * (kTile / 2), o_at = tmem + C::ACC + g * HD;
        uint8_t* const mine = smem + C::OUT + (warp - 4) * 2048;
        float2* const stats = (float2*)(smem + C::STATS);
        // A wait that ran out lets the warp go on without waiting, since the others wait for it at their barriers. Those that the groups share are waits with
        // a limit as well: a warp that never came to know of a unit has left, and does not reach them.
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok) ok = __all_sync(0xffffffffu, wait_barrier(bar, parity, p.status, DEV_ERR_ACC_WAIT));
        };
        uint32_t turns = 0, shared = 0;  // tiles of this group so far; units that all groups have shared
        auto join = [&](uint64_t* bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
            wait(bar, shared & 1u);
            tc_fence_after();
        };
        for (int index = 0; take(index); ++index) {
            if (own && g >= w.n) continue;
            int a_first = w.a_first[0], a_rows = w.a_rows[0], head = w.head[0];
            if (own)
#pragma unroll
                for (int i = 1; i < NG; ++i)
                    if (i == g) {
                        a_first = w.a_first[i];
                        a_rows = w.a_rows[i];
                        head = w.head[i];
                    }
            const bool live = r < a_rows;
            const int grow = w.q_first + a_first + r;  // row of the buffers
            int lo = 0, hi = 0;
            if (live) attn_visible<false>(p, w.q_len, w.k_len, a_first + r, lo, hi);
            float m = -INFINITY, sum = 0.f;
            for (int t = begin; t < w.tiles; t += step, ++turns) {
                const int c_lo = lo - w.first - t * kTile, c_hi = hi - w.first - t * kTile;  // visible columns
                const bool whole = __all_sync(0xffffffffu, c_lo <= 0 && c_hi >= kTile);
                wait(&s_full[g], turns & 1u);
                tc_fence_after();
                uint32_t s[4][16];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld16(s_at + lanes + k * 16, s[k]);
                tc_wait_ld();
                tc_fence_before();
                mbar_arrive(&s_free[g]);
                if (!whole) {  // as bits: eight of them become predicates in one instruction (32 ragged x 512: 30 us, with two comparisons a column 35)
                    const uint64_t seen = bits_between(c_lo, c_hi);
#pragma unroll
                    for (int i = 0; i < kTile; ++i)
                        if (!((uint32_t)(seen >> (i & 32)) & 1u << (i & 31))) s[i >> 4][i & 15] = 0xff800000u;
                }
                auto at = [&](int i) { return __uint_as_float(s[i >> 4][i & 15]); };
                float tops[4] = {at(0), at(1), at(2), at(3)};
#pragma unroll
                for (int i = 4; i < kTile; i += 2) tops[i >> 1 & 3] = max3(tops[i >> 1 & 3], at(i), at(i + 1));
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * p.scale_log2;  // positive scale: the maximum stays the maximum
                float corr = 1.f;
                bool moved = false;
                if (top > m + 8.f || m == -INFINITY) {
                    corr = m == -INFINITY ? 0.f : exp2_fast(m - top);
                    moved = m != -INFINITY;
                    m = top;
                }
                const float ref = m == -INFINITY ? 0.f : m;  // nothing visible yet: every weight is zero
                sum *= corr;
                const F2 scale2 = f2(p.scale_log2, p.scale_log2), ref2 = f2(-ref, -ref);
                uint32_t v[2][16];
                F2 part[2] = {0ull, 0ull};
                // every fourth pair by polynomial where the whole tile is visible (it has no zero)
                auto weights = [&](auto poly) {
#pragma unroll
                    for (int i = 0; i < kTile; i += 2) {
                        const F2 x = fma2(f2(at(i), at(i + 1)), scale2, ref2);
                        float a, b;
                        if (poly.value && i % 8 == 6) {
                            split2(exp2_poly(x), a, b);
                        } else {
                            split2(x, a, b);
                            a = exp2_fast(a);
                            b = exp2_fast(b);
                        }
                        part[i >> 1 & 1] = add2(part[i >> 1 & 1], f2(a, b));
                        v[i >> 5][(i & 31) >> 1] = pack2(a, b);
                    }
                };
                if (whole)
                    weights(std::true_type());
                else
                    weights(std::false_type());
                float parts[4];
                split2(part[0], parts[0], parts[1]);
                split2(part[1], parts[2], parts[3]);
                sum += (parts[0] + parts[1]) + (parts[2] + parts[3]);
                if (t > begin) {  // the product that read the last P, and wrote O
                    wait(&o_full[g], (turns - 1) & 1u);
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll 1
                    for (int k = 0; k < HD / 16; ++k) {
                        uint32_t o[16];
                        tmem_ld16(o_at + lanes + k * 16, o);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                        tmem_st16(o_at + lanes + k * 16, o);
                    }
                }
                tmem_st16(p_at + lanes, v[0]);
                tmem_st16(p_at + lanes + 16, v[1]);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[g]);
            }
            // ---- results of the unit
            const bool any = begin < w.tiles;
            if (any) wait(&o_full[g], (turns - 1) & 1u);
            tc_fence_after();
            const int warp_row = (warp & 3) * 32;
            char* const dst = (char*)(p.out0 + (int64_t)(w.q_first + a_first + warp_row) * p.out0_stride + (int64_t)head * p.hd);
            float weight[NG];  // of each group's O
            if (own) {
                weight[0] = sum > 0.f ? 1.f / sum : 0.f;
            } else {
                stats[g * kStand + r] = make_float2(m, sum);
                join(&joined[0]);
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < NG; ++i) top = fmaxf(top, stats[i * kStand + r].x);
                sum = 0.f;
                m = top;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const float2 x = stats[i * kStand + r];
                    weight[i] = x.x == -INFINITY ? 0.f : exp2_fast(x.x - top);
                    sum = fmaf(x.y, weight[i], sum);
                }
                const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
                for (int i = 0; i < NG; ++i) weight[i] *= inv;
            }
            if (live && p.lse && (own || g == 0)) p.lse[(int64_t)head * p.rows_q + grow] = sum > 0.f ? (m + log2f(sum)) / kLog2e : -INFINITY;
            // a group's own O, or its share of the columns of the joined one
#pragma unroll 1
            for (int c = own ? 0 : 32 * g; c < HD; c += own ? 32 : 32 * NG) {
                float o[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
                auto add = [&](uint32_t from, float f) {
                    uint32_t x[2][16];
                    tmem_ld16(from + c, x[0]);
                    tmem_ld16(from + c + 16, x[1]);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = fmaf(__uint_as_float(x[i >> 4][i & 15]), f, o[i]);
                };
                if (own) {
                    if (any) add(o_at + lanes, weight[0]);
                } else {
#pragma unroll
                    for (int i = 0; i < NG; ++i)
                        if (w.tiles > i) add(tmem + lanes + C::ACC + i * HD, weight[i]);
                }
                uint4 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = make_uint4(pack2(o[8 * i], o[8 * i + 1]), pack2(o[8 * i + 2], o[8 * i + 3]), pack2(o[8 * i + 4], o[8 * i + 5]), pack2(o[8 * i + 6], o[8 * i + 7]));
                store_rows(mine, v, dst + c * 2, p.out0_stride * 2, a_rows - warp_row, (p.hd - c) / 8);
            }
            tc_fence_before();
            if (!own) {  // every group has read every O, and the statistics
                join(&joined[1]);
                ++shared;
            }
            if (any) mbar_arrive(&o_free[g]);
        }
    }
    tc_fence_before();
    if (__syncthreads_or(!ok)) let_land();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

// slots of a chunk, where a block of 128 queries has heads / parts of them; a chunk without an end is as good as none
int chunk_slots(const AttnCall& c, int heads, int parts) {
    return c.chunk == 0 ? 0 : (int)std::min<int64_t>(std::max<int64_t>((int64_t)c.chunk / kStand * heads / parts, 1), 1 << 28);
}

template <int HD>
int run(AttnDev& p, const AttnCall& c, int num_sms, cudaStream_t s) {
    using C = Cfg<HD>;
    const int G = c.heads / c.kv_heads;
    const int64_t blocks = (c.max_q + kStand - 1) / kStand, all = blocks * c.n_seqs * c.heads;
    // Units to themselves where every group of every SM gets four, counted by the bounds (ragged sequences have fewer: 32 x 512 2.6), us (one unit
    // at a time against units of their own): 1 x 8 192, 28 heads of 128 467 against 411; 8 x 4 096, 14 heads of 64 390 against 319; 32 ragged x 512 of them
    // 41 against 34; 3 x 2 777 of them in chunks of 1 024 44 against 75; 1 x 1 000 of them 16 against 37.
    p.parts = all <= 4 * C::GROUPS * num_sms ? 1 : C::GROUPS;
    const int64_t n = std::min<int64_t>(c.n_seqs, c.rows_q);  // sequences with rows
    const int64_t units = std::min((blocks * G + p.parts - 1) / p.parts * c.n_seqs, blocks_of_rows(c, c.max_q, c.rows_q) * G / p.parts + n) * c.kv_heads;
    const unsigned grid = set_units(p, units, num_sms);
    p.chunk_slots = chunk_slots(c, G, p.parts);
    p.by_fast = FastDiv::of(c.kv_heads);
    p.by_parts = FastDiv::of(p.parts);
    const cudaError_t e = allow_shared<k_attn_fwd<HD>>(C::SMEM);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_k(k_attn_fwd<HD>, dim3(grid), dim3(C::THREADS), (size_t)C::SMEM, s, false, p);
}

}  // namespace

AttnDev attn_dev(const AttnCall& c) {
    AttnDev p;
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
    p.group = c.heads / c.kv_heads;
    p.by_group = FastDiv::of(p.group);
    p.by_chunk = FastDiv::of(c.chunk > 0 ? c.chunk : 1);
    p.by_fast = p.by_parts = FastDiv::of(1);
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

int64_t blocks_of_rows(const AttnCall& c, int most, int64_t rows) {
    return std::min((int64_t)((most + kStand - 1) / kStand) * c.n_seqs, rows / kStand + std::min<int64_t>(c.n_seqs, rows));
}
unsigned set_units(AttnDev& p, int64_t units, int num_sms) {
    p.units = (int)std::min(units, kMostUnits - 1);
    const int grid = std::min(p.units, num_sms), groups = (p.n_seqs + 31) / 32;
    p.most_levels = groups <= 1 ? INT32_MAX : std::max(32, 4 * (p.units / grid)) / groups;  // 32 sequences are one order either way
    return (unsigned)grid;
}
bool attention_forward_fits(const AttnCall& c) { return blocks_of_rows(c, c.max_q, c.rows_q) * c.heads < kMostUnits; }

bool map_heads(CUtensorMap* tm, const bf16* x, int64_t rows, int64_t stride, int heads, int hd, int box) {
    return make_tmap_2d(nullptr, tm, x, (uint64_t)rows, (uint64_t)hd, (uint64_t)stride, (uint32_t)box, (uint32_t)heads, (uint32_t)hd);
}

int launch_attention_train_forward(const AttnCall& c, int num_sms, cudaStream_t s) {
    if (c.n_seqs == 0 || c.max_q == 0 || c.rows_q == 0) return 0;
    AttnDev p = attn_dev(c);
    if (!map_heads(&p.tmA[0], c.q, c.rows_q, c.q_stride, c.heads, c.hd, kStand)) return -1000;
    p.tm[0] = p.tm[1] = p.tmA[0];  // no keys at all: any valid map, none of its rows is read
    if (c.rows_k > 0 && c.max_k > 0 &&
        (!map_heads(&p.tm[0], c.k, c.rows_k, c.k_stride, c.kv_heads, c.hd, kTile) || !map_heads(&p.tm[1], c.v, c.rows_k, c.v_stride, c.kv_heads, c.hd, kTile)))
        return -1000;
    p.out0 = c.out;
    p.out0_stride = c.out_stride;
    return c.hd <= 64 ? run<64>(p, c, num_sms, s) : run<128>(p, c, num_sms, s);
}

}  // namespace tffn
