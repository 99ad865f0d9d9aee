// Attention backward on the tensor cores: two kernels, each result with one owner and one order of its sums.
//
// attn_tc_dkv_kernel: a block owns 128 keys of one key head and walks over the queries (of all query heads that read
// it) in tiles of 128.  Everything is taken across, keys as rows: S' = K Q' and dP' = V dO' into tensor memory; the
// weights P' = 2^(S' - lse) go back as bf16 over S' and dS' = P' (dP' - delta) over dP', operands of dV += P' dO and
// dK += dS' Q.  lse and delta belong to columns and come out of shared memory.
// attn_tc_dq_kernel: a block owns 128 queries and walks over the keys, queries as rows: S = Q K', dP = dO V',
// dQ += dS K.  It works S and dP out a second time (7 products in all instead of 5), for which no sum over blocks is
// needed: no atomics, no fp32 gradient in memory, the same bits every run.
//
// Two teams of 128 threads have half of a step's columns each, all 128 rows.  The products of one part of a step run
// under the exponentials of another: P' and dS' are handed over apart, and the scores are taken a step (dkv) or two
// (dq) ahead.  Heads of 128 channels: steps of 128 columns, one block an SM, whose tensor memory they fill.  Heads of 64:
// steps of 64 columns and two blocks an SM, whose steps fall under one another's.
//
// 8 heads of 128 channels, 2 key heads, 12288 cells, causal: dkv 487 us, dq 332 (1.32 PFLOP/s over the
// seven products); the tensor pipe is busy 68 and 70 % of the time.  2 x 8 heads of 64 on 64^2 cells: 180 and 140 us; issue slots
// half full, the tensor pipe 38 %.
#include "attention_tc.cuh"

namespace dcb
{
namespace
{

template <int D>
struct AbShape
{
    static constexpr int BLOCKS = D == 64 ? 2 : 1;        // an SM
    static constexpr int STEP = D == 64 ? 64 : 128;       // columns
    static constexpr int MINE = STEP / 2;                 // of a team
    static constexpr uint32_t COLUMNS = 512 / BLOCKS;     // of tensor memory
    static constexpr int TEAM_REGS = BLOCKS == 2 ? 104 : AT_TEAM_REGS;
    static constexpr int OTHER_REGS = BLOCKS == 2 ? 32 : AT_OTHER_REGS;
    static constexpr uint32_t BYTES = AtTile<D>::HALF * (STEP / 64); // of a step's operand
    static constexpr uint32_t A_SLOTS = D == 128 ? 3 : 4; // Q (dkv) or K (dq)
    static constexpr uint32_t B_SLOTS = D == 128 ? 2 : 3; // dO (dkv) or V (dq)
    static constexpr uint32_t OWN_AT = 0;                 // K, V (dkv) or Q, dO (dq): 128 cells each
    static constexpr uint32_t A_AT = 2 * AtTile<D>::BYTES;
    static constexpr uint32_t B_AT = A_AT + A_SLOTS * BYTES;
    static constexpr uint32_t STATS_AT = B_AT + B_SLOTS * BYTES; // dkv: lse, delta of a dO slot
    static constexpr uint32_t BARS_AT = STATS_AT + B_SLOTS * 8 * STEP;
    static constexpr uint32_t SMEM = BARS_AT + 256;
    // columns: dkv S, dP, dV, dK; dq S twice, dP, dQ
    static constexpr uint32_t DKV_DP = STEP, DKV_DV = 2 * STEP, DKV_DK = 2 * STEP + D;
    static constexpr uint32_t DQ_DP = 2 * STEP, DQ_DQ = 3 * STEP;
};
template <int D>
constexpr bool ab_fits = AbShape<D>::DKV_DK + D <= AbShape<D>::COLUMNS && AbShape<D>::DQ_DQ + D <= AbShape<D>::COLUMNS
                         && AbShape<D>::BLOCKS * (AbShape<D>::SMEM + 1024) <= 228 * 1024;
static_assert(ab_fits<64> && ab_fits<128>, "tensor memory of a block, shared memory of an SM's blocks");
static_assert(2 * AbShape<64>::TEAM_REGS + AbShape<64>::OTHER_REGS <= 3 * 80, "registers of two blocks");

struct AbBars
{
    uint64_t own_full, a_full[4], a_empty[4], b_full[4], b_empty[4], s_full[2], dp_full, p_ready, ds_ready, fin;
    uint32_t tmem;
    int give_up;
};
static_assert(sizeof(AbBars) <= 256, "the barriers' room");

template <uint32_t COLUMNS>
__device__ __forceinline__ void ab_init(AbBars& b, int warp)
{
    if (threadIdx.x == 0)
    {
        mbar_init(&b.own_full, 1);
        for (int s = 0; s < 4; ++s)
        {
            mbar_init(&b.a_full[s], 1), mbar_init(&b.a_empty[s], 1);
            mbar_init(&b.b_full[s], 1), mbar_init(&b.b_empty[s], 1);
        }
        mbar_init(&b.s_full[0], 1), mbar_init(&b.s_full[1], 1);
        mbar_init(&b.dp_full, 1), mbar_init(&b.fin, 1);
        mbar_init(&b.p_ready, 8), mbar_init(&b.ds_ready, 8);
        b.give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == AT_MMA_WARP)
        at_tmem_alloc<COLUMNS>(&b.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
}

// The block gave up: the products that were issued end before the tensor memory goes back.
__device__ __forceinline__ void ab_drain_products(AbBars& b, uint32_t elected)
{
    int none = 0;
    at_commit(&b.fin, elected);
    mbar_wait_t<20>(&b.fin, 0, &none);
}

// d += W B over a step's cells: a team's half of W lies at the start of its scores' columns, two cells to a column.
template <int D>
__device__ __forceinline__ void ab_weigh(uint32_t d, uint32_t w, uint32_t b, uint32_t n, bool first, uint32_t elected)
{
    constexpr int MINE = AbShape<D>::MINE;
    const uint32_t idesc = at_idesc(n, false, false);
#pragma unroll
    for (int k = 0; k < 2 * MINE / 16; ++k)
    {
        const int team = k / (MINE / 16), in_team = k % (MINE / 16);
        const uint64_t db = AtTile<D>::along(b + k / 4 * AtTile<D>::HALF) + k % 4 * 2;
        at_mma_ts(d, w + team * MINE + in_team * 8, db, idesc, !(first && k == 0), elected);
    }
}

template <int N>
__device__ __forceinline__ void ab_fetch(uint32_t taddr, float (&v)[N])
{
#pragma unroll
    for (int c = 0; c < N; c += 32)
        at_tmem_ld32(taddr + c, v + c);
}

template <int N>
__device__ __forceinline__ void ab_put(uint32_t taddr, const uint32_t (&v)[N])
{
    if constexpr (N == 32)
        at_tmem_st32(taddr, v);
    else
        at_tmem_st16(taddr, v);
}

template <int D>
__global__ void __launch_bounds__(AT_THREADS, AbShape<D>::BLOCKS)
    attn_tc_dkv_kernel(const __grid_constant__ AttnProblem p, const __grid_constant__ AtMaps maps)
{
    using S = AbShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    AbBars& b = *reinterpret_cast<AbBars*>(smem + S::BARS_AT);
    const int warp = __shfl_sync(~0u, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int* give_up = &b.give_up;
    if (at_misplaced(base))
        return;

    const int tiles_k = attn_tiles(p.sk, AT_TILE);
    long long at;
    const int tile = at_block(p.causal, tiles_k, (long long) p.n * p.kv_heads * p.q_splits, &at); // the first keys' are longest
    const int split = (int) (at % p.q_splits);
    const long long nh = at / p.q_splits, n = nh / p.kv_heads;
    const int head = (int) (nh - n * p.kv_heads);
    const int j0 = tile * AT_TILE;
    ab_init<S::COLUMNS>(b, warp);
    const uint32_t tmem = __shfl_sync(~0u, b.tmem, 0); // known to be uniform
    const float* stats = p.stats;
    wait_for_previous_kernel(stats);
    const AttnCells q(p.q_side, n, p.sq), kv(p.kv_side, n, p.sk);
    // a key is seen from this row of the queries on
    const auto first_row = [&](int r) {
        return r >= kv.count ? q.count : p.causal ? q.before((long long) kv.cell(r) - p.offset) : 0;
    };
    // the walk: steps of queries from t0 on, of every query head of the group
    const int t0 = first_row(j0) / S::STEP;
    const int per_head = max(0, attn_tiles(q.count, S::STEP) - t0);
    const long long all = j0 < kv.count ? (long long) per_head * p.group : 0;
    const int lo = (int) (all * split / p.q_splits), steps = (int) (all * (split + 1) / p.q_splits) - lo;
    bool ok = true;
    const uint32_t s_at = tmem, dp_at = tmem + S::DKV_DP, dv_at = tmem + S::DKV_DV, dk_at = tmem + S::DKV_DK;

    if (warp >= AT_MMA_WARP)
    {
        at_fewer_registers<S::OTHER_REGS>();
        if (warp == AT_TMA_WARP)
        {
            if (lane == 0 && steps > 0)
            {
                mbar_expect_tx(&b.own_full, 2 * AtTile<D>::BYTES);
                at_tma_tile<D>(base + S::OWN_AT, &maps.k, j0, head, (int) n, &b.own_full);
                at_tma_tile<D>(base + S::OWN_AT + AtTile<D>::BYTES, &maps.v, j0, head, (int) n, &b.own_full);
                AtRing ra, rb;
                for (int u = 0; u < steps && ok; ++u)
                {
                    const int g = (lo + u) / per_head, i0 = (t0 + (lo + u) - g * per_head) * S::STEP;
                    const int q_head = head * p.group + g;
                    if (ra.lap > 0)
                        ok = mbar_wait_t<20>(&b.a_empty[ra.slot], (ra.lap - 1) & 1, give_up);
                    if (!ok)
                        break;
                    mbar_expect_tx(&b.a_full[ra.slot], S::BYTES);
                    at_tma_cells<D, S::STEP>(base + S::A_AT + ra.slot * S::BYTES, &maps.q, i0, q_head, (int) n,
                                             &b.a_full[ra.slot]);
                    ra.next(S::A_SLOTS);
                    if (rb.lap > 0)
                        ok = mbar_wait_t<20>(&b.b_empty[rb.slot], (rb.lap - 1) & 1, give_up);
                    if (!ok)
                        break;
                    mbar_expect_tx(&b.b_full[rb.slot], S::BYTES + 8 * S::STEP);
                    at_tma_cells<D, S::STEP>(base + S::B_AT + rb.slot * S::BYTES, &maps.d_o, i0, q_head, (int) n,
                                             &b.b_full[rb.slot]);
                    const float* row = stats + (n * p.q_heads + q_head) * p.stats_pitch + i0;
                    at_bulk(base + S::STATS_AT + rb.slot * 8 * S::STEP, row, 4 * S::STEP, &b.b_full[rb.slot]);
                    at_bulk(base + S::STATS_AT + rb.slot * 8 * S::STEP + 4 * S::STEP,
                            row + (long long) p.n * p.q_heads * p.stats_pitch, 4 * S::STEP, &b.b_full[rb.slot]);
                    rb.next(S::B_SLOTS);
                }
                if (!ok || *give_up)
                {
                    int none = 0;
                    mbar_wait_t<20>(&b.own_full, 0, &none);
                    at_drain(b.a_full, S::A_SLOTS, ra);
                    at_drain(b.b_full, S::B_SLOTS, rb);
                }
            }
        }
        else if (warp == AT_MMA_WARP)
        {
            if (steps > 0)
            {
                const uint32_t elected = at_elect();
                const int ksteps = (p.d + 15) / 16;
                const uint32_t width = (uint32_t) ksteps * 16;
                const uint32_t k_at = base + S::OWN_AT, v_at = k_at + AtTile<D>::BYTES;
                AtRing ra, rb; // of the next tiles to wait for
                uint32_t q_slot = 0, o_slot = 0;
                const auto scores = [&] {
                    ok = ok && at_warp_wait(&b.a_full[ra.slot], ra.lap & 1, give_up);
                    if (!ok)
                        return;
                    tc_fence_after();
                    at_scores<D, S::STEP>(s_at, k_at, base + S::A_AT + ra.slot * S::BYTES, ksteps, elected);
                    at_commit(&b.s_full[0], elected);
                    ra.next(S::A_SLOTS);
                };
                const auto weight_grads = [&] {
                    ok = ok && at_warp_wait(&b.b_full[rb.slot], rb.lap & 1, give_up);
                    if (!ok)
                        return;
                    tc_fence_after();
                    at_scores<D, S::STEP>(dp_at, v_at, base + S::B_AT + rb.slot * S::BYTES, ksteps, elected);
                    at_commit(&b.dp_full, elected);
                    rb.next(S::B_SLOTS);
                };
                ok = at_warp_wait(&b.own_full, 0, give_up);
                scores();
                weight_grads();
                for (int u = 0; u < steps && ok; ++u)
                {
                    ok = at_warp_wait(&b.p_ready, u & 1, give_up);
                    if (!ok)
                        break;
                    tc_fence_after();
                    ab_weigh<D>(dv_at, s_at, base + S::B_AT + o_slot * S::BYTES, width, u == 0, elected);
                    if (u + 1 < steps)
                        scores();
                    ok = ok && at_warp_wait(&b.ds_ready, u & 1, give_up);
                    if (!ok)
                        break;
                    tc_fence_after();
                    ab_weigh<D>(dk_at, dp_at, base + S::A_AT + q_slot * S::BYTES, width, u == 0, elected);
                    at_commit(&b.a_empty[q_slot], elected);
                    at_commit(&b.b_empty[o_slot], elected);
                    q_slot = q_slot + 1 == S::A_SLOTS ? 0 : q_slot + 1;
                    o_slot = o_slot + 1 == S::B_SLOTS ? 0 : o_slot + 1;
                    if (u + 1 < steps)
                        weight_grads();
                }
                if (ok)
                    at_commit(&b.fin, elected);
                else
                    ab_drain_products(b, elected);
            }
        }
    }
    else
    {
        at_more_registers<S::TEAM_REGS>();
        const int team = warp >> 2;
        const uint32_t lanes = (uint32_t) (warp & 3) << 21;
        const int row = j0 + (threadIdx.x & 127), j = row < kv.count ? kv.cell(row) : -1, from = first_row(row);
        const uint32_t s_mine = s_at + lanes + S::MINE * team, dp_mine = dp_at + lanes + S::MINE * team;
        AtRing rb;
        for (int u = 0; u < steps; ++u)
        {
            const int g = (lo + u) / per_head, i0 = (t0 + (lo + u) - g * per_head) * S::STEP + S::MINE * team;
            const float* lse = reinterpret_cast<const float*>(smem + S::STATS_AT + rb.slot * 8 * S::STEP) + S::MINE * team;
            ok = at_warp_wait(&b.b_full[rb.slot], rb.lap & 1, give_up)
                 && at_warp_wait(&b.s_full[0], u & 1, give_up);
            if (!ok)
                break;
            rb.next(S::B_SLOTS);
            tc_fence_after();
            float w[S::MINE];
            ab_fetch<S::MINE>(s_mine, w);
            at_tmem_wait_ld();
            // this key is seen by the cells from `first` on of this team's
            const int first = j < 0 ? 0 : from - i0;
            const bool cut = __any_sync(~0u, first > 0);
#pragma unroll
            for (int c = 0; c < S::MINE; c += 4)
            {
                float l[4];
                load_elems<4>(lse + c, l);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[c + e] = at_exp2(fmaf(w[c + e], p.scale, -l[e]));
            }
            if (cut)
            {
#pragma unroll
                for (int c = 0; c < S::MINE; ++c)
                    w[c] = c >= first ? w[c] : 0.f;
            }
            {
                uint32_t packed[S::MINE / 2];
#pragma unroll
                for (int c = 0; c < S::MINE / 2; ++c)
                    packed[c] = pack_bf16(w[2 * c], w[2 * c + 1]);
                ab_put<S::MINE / 2>(s_mine, packed);
            }
            at_tmem_wait_st();
            at_warp_arrive(&b.p_ready, lane);

            ok = at_warp_wait(&b.dp_full, u & 1, give_up);
            if (!ok)
                break;
            tc_fence_after();
            float d[S::MINE];
            ab_fetch<S::MINE>(dp_mine, d);
            at_tmem_wait_ld();
            const float* delta = lse + S::STEP;
            uint32_t packed[S::MINE / 2];
#pragma unroll
            for (int c = 0; c < S::MINE; c += 4)
            {
                float l[4];
                load_elems<4>(delta + c, l);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    d[c + e] = w[c + e] * (d[c + e] - l[e]);
                packed[c / 2] = pack_bf16(d[c], d[c + 1]);
                packed[c / 2 + 1] = pack_bf16(d[c + 2], d[c + 3]);
            }
            if (cut)
            {
#pragma unroll
                for (int c = 0; c < S::MINE / 2; ++c)
                    packed[c] = 2 * c >= first ? packed[c] : 2 * c + 1 >= first ? packed[c] & 0xffff0000u : 0u;
            }
            ab_put<S::MINE / 2>(dp_mine, packed);
            at_tmem_wait_st();
            at_warp_arrive(&b.ds_ready, lane);
        }
        if (ok && steps > 0)
            ok = at_warp_wait(&b.fin, 0, give_up);
        tc_fence_after();
        if (ok)
        {
            const long long part = (long long) p.n * p.kv_heads * p.d * p.sk * split;
            if (team == 0)
                at_store(p.dv, p.q_splits > 1 ? p.part_dv + part : nullptr, nh, n, head, p.d, j, p.sk, 1.f, false,
                         steps == 0, dv_at + lanes, 0, D);
            else
                at_store(p.dk, p.q_splits > 1 ? p.part_dk + part : nullptr, nh, n, head, p.d, j, p.sk,
                         p.scale / ATTN_LOG2E, false, steps == 0, dk_at + lanes, 0, D);
        }
    }
    at_finish<S::COLUMNS>(ok, warp, lane, tmem);
}

template <int D>
__global__ void __launch_bounds__(AT_THREADS, AbShape<D>::BLOCKS)
    attn_tc_dq_kernel(const __grid_constant__ AttnProblem p, const __grid_constant__ AtMaps maps)
{
    using S = AbShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    AbBars& b = *reinterpret_cast<AbBars*>(smem + S::BARS_AT);
    const int warp = __shfl_sync(~0u, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int* give_up = &b.give_up;
    if (at_misplaced(base))
        return;

    const int tiles_q = attn_tiles(p.sq, AT_TILE);
    long long at;
    const int tile = tiles_q - 1 - at_block(p.causal, tiles_q, (long long) p.n * p.q_heads * p.kv_splits, &at);
    const int split = (int) (at % p.kv_splits);
    const long long nh = at / p.kv_splits, n = nh / p.q_heads;
    const int head = (int) (nh - n * p.q_heads), kv_head = head / p.group;
    const int i0 = tile * AT_TILE;

    ab_init<S::COLUMNS>(b, warp);
    const uint32_t tmem = __shfl_sync(~0u, b.tmem, 0); // known to be uniform
    const float* stats = p.stats;
    wait_for_previous_kernel(stats);
    const AttnCells q(p.q_side, n, p.sq), kv(p.kv_side, n, p.sk);
    const int steps_k = attn_tiles(kv.count, S::STEP);
    const int lo = (int) ((long long) steps_k * split / p.kv_splits);
    const int hi = min((int) ((long long) steps_k * (split + 1) / p.kv_splits),
                       attn_tiles(attn_limit(p, q, kv, min(i0 + AT_TILE, q.count) - 1), S::STEP));
    const int steps = i0 < q.count ? max(0, hi - lo) : 0;
    bool ok = true;
    const uint32_t s_at = tmem, dp_at = tmem + S::DQ_DP, dq_at = tmem + S::DQ_DQ;

    if (warp >= AT_MMA_WARP)
    {
        at_fewer_registers<S::OTHER_REGS>();
        if (warp == AT_TMA_WARP)
        {
            if (lane == 0 && steps > 0)
            {
                mbar_expect_tx(&b.own_full, 2 * AtTile<D>::BYTES);
                at_tma_tile<D>(base + S::OWN_AT, &maps.q, i0, head, (int) n, &b.own_full);
                at_tma_tile<D>(base + S::OWN_AT + AtTile<D>::BYTES, &maps.d_o, i0, head, (int) n, &b.own_full);
                AtRing ra, rb;
                for (int u = 0; u < 2 * steps && ok; ++u) // K and V in turn
                {
                    AtRing& r = u & 1 ? rb : ra;
                    const uint32_t slots = u & 1 ? S::B_SLOTS : S::A_SLOTS;
                    uint64_t *full = u & 1 ? b.b_full : b.a_full, *empty = u & 1 ? b.b_empty : b.a_empty;
                    if (r.lap > 0)
                        ok = mbar_wait_t<20>(&empty[r.slot], (r.lap - 1) & 1, give_up);
                    if (!ok)
                        break;
                    mbar_expect_tx(&full[r.slot], S::BYTES);
                    at_tma_cells<D, S::STEP>(base + (u & 1 ? S::B_AT : S::A_AT) + r.slot * S::BYTES,
                                             u & 1 ? &maps.v : &maps.k, (lo + (u >> 1)) * S::STEP, kv_head, (int) n,
                                             &full[r.slot]);
                    r.next(slots);
                }
                if (!ok || *give_up)
                {
                    int none = 0;
                    mbar_wait_t<20>(&b.own_full, 0, &none);
                    at_drain(b.a_full, S::A_SLOTS, ra);
                    at_drain(b.b_full, S::B_SLOTS, rb);
                }
            }
        }
        else if (warp == AT_MMA_WARP)
        {
            if (steps > 0)
            {
                const uint32_t elected = at_elect();
                const int ksteps = (p.d + 15) / 16;
                const uint32_t width = (uint32_t) ksteps * 16;
                const uint32_t q_at = base + S::OWN_AT, do_at = q_at + AtTile<D>::BYTES;
                AtRing ra, rb; // of the next tiles to wait for
                uint32_t k_slot = 0;
                int ahead = 0; // scores taken so far
                const auto scores = [&] {
                    ok = ok && at_warp_wait(&b.a_full[ra.slot], ra.lap & 1, give_up);
                    if (!ok)
                        return;
                    tc_fence_after();
                    at_scores<D, S::STEP>(s_at + S::STEP * (ahead & 1), q_at, base + S::A_AT + ra.slot * S::BYTES, ksteps, elected);
                    at_commit(&b.s_full[ahead & 1], elected);
                    ++ahead;
                    ra.next(S::A_SLOTS);
                };
                const auto weight_grads = [&] {
                    ok = ok && at_warp_wait(&b.b_full[rb.slot], rb.lap & 1, give_up);
                    if (!ok)
                        return;
                    tc_fence_after();
                    at_scores<D, S::STEP>(dp_at, do_at, base + S::B_AT + rb.slot * S::BYTES, ksteps, elected);
                    at_commit(&b.dp_full, elected);
                    at_commit(&b.b_empty[rb.slot], elected);
                    rb.next(S::B_SLOTS);
                };
                ok = at_warp_wait(&b.own_full, 0, give_up);
                scores();
                weight_grads();
                if (steps > 1)
                    scores();
                for (int u = 0; u < steps && ok; ++u)
                {
                    ok = at_warp_wait(&b.ds_ready, u & 1, give_up);
                    if (!ok)
                        break;
                    tc_fence_after();
                    ab_weigh<D>(dq_at, dp_at, base + S::A_AT + k_slot * S::BYTES, width, u == 0, elected);
                    at_commit(&b.a_empty[k_slot], elected);
                    k_slot = k_slot + 1 == S::A_SLOTS ? 0 : k_slot + 1;
                    if (u + 1 < steps)
                        weight_grads();
                    if (u + 2 < steps)
                        scores();
                }
                if (ok)
                    at_commit(&b.fin, elected);
                else
                    ab_drain_products(b, elected);
            }
        }
    }
    else
    {
        at_more_registers<S::TEAM_REGS>();
        const int team = warp >> 2;
        const uint32_t lanes = (uint32_t) (warp & 3) << 21;
        const int row0 = i0 + (warp & 3) * 32, r = row0 + lane;
        const int i = r < q.count ? q.cell(r) : -1, limit = attn_limit(p, q, kv, r);
        const int open = max(0, attn_limit(p, q, kv, row0) - lo * S::STEP) / S::STEP; // steps that all its rows see whole
        const uint32_t dp_mine = dp_at + lanes + S::MINE * team;
        const float* row = stats + nh * p.stats_pitch + r; // up to a multiple of 128 cells
        const float lse = row[0], delta = row[(long long) p.n * p.q_heads * p.stats_pitch];
        for (int u = 0; u < steps; ++u)
        {
            const int j0 = (lo + u) * S::STEP + S::MINE * team;
            const uint32_t s_mine = s_at + lanes + S::STEP * (u & 1) + S::MINE * team;
            ok = at_warp_wait(&b.s_full[u & 1], (u >> 1) & 1, give_up);
            if (!ok)
                break;
            tc_fence_after();
            float w[S::MINE];
            ab_fetch<S::MINE>(s_mine, w);
            at_tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < S::MINE; ++c)
                w[c] = at_exp2(fmaf(w[c], p.scale, -lse));
            ok = at_warp_wait(&b.dp_full, u & 1, give_up);
            if (!ok)
                break;
            tc_fence_after();
            float d[S::MINE];
            ab_fetch<S::MINE>(dp_mine, d);
            at_tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < S::MINE; ++c)
                d[c] = w[c] * (d[c] - delta);
            if (u >= open)
            {
                uint32_t see[S::MINE / 32];
#pragma unroll
                for (int k = 0; k < S::MINE / 32; ++k)
                    see[k] = at_up_to(limit - 1 - j0, k);
#pragma unroll
                for (int c = 0; c < S::MINE; ++c)
                    d[c] = see[c >> 5] >> (c & 31) & 1 ? d[c] : 0.f;
            }
            uint32_t packed[S::MINE / 2];
#pragma unroll
            for (int c = 0; c < S::MINE / 2; ++c)
                packed[c] = pack_bf16(d[2 * c], d[2 * c + 1]);
            ab_put<S::MINE / 2>(dp_mine, packed);
            at_tmem_wait_st();
            at_warp_arrive(&b.ds_ready, lane);
        }
        if (ok && steps > 0)
            ok = at_warp_wait(&b.fin, 0, give_up);
        tc_fence_after();
        if (ok)
        {
            float* part = p.kv_splits > 1 ? p.part_dq + (long long) split * p.n * p.q_heads * p.d * p.sq : nullptr;
            at_store(p.dq, part, nh, n, head, p.d, i, p.sq, p.scale / ATTN_LOG2E, lse == INFINITY, steps == 0,
                     dq_at + lanes, team * (D / 2), (team + 1) * (D / 2));
        }
    }
    at_finish<S::COLUMNS>(ok, warp, lane, tmem);
}

template <int D>
int32_t ab_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream)
{
    const long long dkv = (long long) p.n * p.kv_heads * attn_tiles(p.sk, AT_TILE) * p.q_splits;
    const long long dq = (long long) p.n * p.q_heads * attn_tiles(p.sq, AT_TILE) * p.kv_splits;
    DCB_REQUIRE(dkv < (1ll << 31) && dq < (1ll << 31), "too many tiles");
    if (int32_t e = allow_dynamic_smem((const void*) attn_tc_dkv_kernel<D>, AbShape<D>::SMEM))
        return e;
    if (int32_t e = allow_dynamic_smem((const void*) attn_tc_dq_kernel<D>, AbShape<D>::SMEM))
        return e;
    DCB_CUDA_TRY(launch_overlapped(attn_tc_dkv_kernel<D>, dim3((unsigned) dkv), AT_THREADS, AbShape<D>::SMEM, stream, p, maps));
    DCB_CUDA_TRY(launch_overlapped(attn_tc_dq_kernel<D>, dim3((unsigned) dq), AT_THREADS, AbShape<D>::SMEM, stream, p, maps));
    return DCB_OK;
}

} // namespace

int32_t attn_tc_bwd_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream)
{
    return p.d <= 64 ? ab_launch<64>(p, maps, stream) : ab_launch<128>(p, maps, stream);
}

int32_t attn_tc_bwd_status(bool* gave_up)
{
    return at_read_status(gave_up);
}

} // namespace dcb
