// Attention forward on the tensor cores.
//
// A block has two tiles of 128 query cells of one head, each with a team of 128 threads, one row a thread, and walks over
// the keys, 64 at a step.  A step's scores S = Q K' arrive in tensor memory, the team turns them into weights, writes them
// back as bf16 over the scores, and the tensor cores add O += P V.  With 128 channels a team's scores have two places: the
// tensor cores take the next step's while the threads work on this one's.  With 64 there are two blocks an SM instead,
// whose steps fall under one another's.  (One place of 128 columns and one block: teams waited for products a third of
// the time, 4 x 4096 cells, 8 heads of 64 channels 257 us.)  A row's weights are powers of two about a maximum that is
// renewed only when it has grown by more than 2^8 since; then the thread scales its row of O.  (The sums are exact about
// any base that keeps them in range.)
//
// 64 channels, 4 x 8 heads on 64^2 cells: 208 us (660 TFLOP/s); bound by the threads that make weights: half of the issue
// slots, 56 % of the exponentials' unit, hand-overs between.  128 channels, 8 heads on 12288 cells: 611 us (1010 TFLOP/s),
// causal 309 us; the tensor pipe and the exponentials at half each.
//
// Few queries of such heads, many keys (APART): both teams have the same 128 queries and a part of the keys each.
#include "attention_tc.cuh"

namespace dcb
{

namespace
{

constexpr float AF_GROWTH = 8.f;

// Heads of 64 channels: two blocks an SM, of half its tensor memory each, so that an SM sub-core has four rows' warps;
// a team has one place for scores then.  128 channels: one block.
template <int D, bool APART>
struct AfShape
{
    static constexpr int BLOCKS = D == 64 && !APART ? 2 : 1; // an SM
    static constexpr int PLACES = BLOCKS == 2 ? 1 : 2;  // for 64 columns of a team's scores
    static constexpr uint32_t O_AT = 2 * PLACES * 64;   // column of O, D a team
    static constexpr uint32_t SLOTS = D == 128 ? 5 : BLOCKS == 2 ? 4 : 8; // of K and V tiles in turn
    static constexpr uint32_t COLUMNS = 512 / BLOCKS;
    // registers: 3 x 80 (two blocks) or 3 x 168 at launch
    static constexpr int TEAM_REGS = BLOCKS == 2 ? 104 : AT_TEAM_REGS;
    static constexpr int OTHER_REGS = BLOCKS == 2 ? 32 : AT_OTHER_REGS;
    static constexpr uint32_t Q_AT = 0;
    static constexpr uint32_t RING_AT = 2 * AtTile<D>::BYTES;
    static constexpr uint32_t BARS_AT = RING_AT + SLOTS * AtTile<D>::BYTES;
    static constexpr uint32_t SMEM = BARS_AT + 256;
};
template <int D, bool APART>
constexpr bool af_fits = AfShape<D, APART>::O_AT + 2 * D <= AfShape<D, APART>::COLUMNS
                         && AfShape<D, APART>::BLOCKS * (AfShape<D, APART>::SMEM + 1024) <= 228 * 1024;
static_assert(af_fits<64, false> && af_fits<64, true> && af_fits<128, false>,
              "tensor memory of a block, shared memory of an SM's blocks");
static_assert(2 * AfShape<64, false>::TEAM_REGS + AfShape<64, false>::OTHER_REGS <= 3 * 80, "registers of two blocks");

struct AfBars
{
    uint64_t q_full, full[8], empty[8], s_full[2][2], p_ready[2][2], o_done[2], fin[2];
    uint32_t tmem;
    int give_up;
};
static_assert(sizeof(AfBars) <= 256, "the barriers' room");

template <int D, bool APART>
__global__ void __launch_bounds__(AT_THREADS, AfShape<D, APART>::BLOCKS)
    attn_tc_fwd_kernel(const __grid_constant__ AttnProblem p, const __grid_constant__ AtMaps maps)
{
    using S = AfShape<D, APART>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    AfBars& b = *reinterpret_cast<AfBars*>(smem + S::BARS_AT);
    const int warp = __shfl_sync(~0u, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int* give_up = &b.give_up;
    if (at_misplaced(base))
        return;

    const int blocks_q = APART ? 1 : attn_tiles(p.sq, 2 * AT_TILE);
    const int splits = APART ? p.kv_splits / 2 : p.kv_splits;
    long long at;
    const int block_q = blocks_q - 1 - at_block(p.causal, blocks_q, (long long) p.n * p.q_heads * splits, &at);
    const int split = (int) (at % splits);
    const long long nh = at / splits, n = nh / p.q_heads;
    const int head = (int) (nh - n * p.q_heads), kv_head = head / p.group;
    const int i0 = block_q * 2 * AT_TILE;
    // K and V tiles in the order that they are needed in: number of team t's, of the j-th tile
    const auto k_number = [&](int t, int j) { return (uint32_t) (APART ? 4 * j + t : 2 * j); };
    const auto v_number = [&](int t, int j) { return (uint32_t) (APART ? 4 * j + 2 + t : 2 * j + 1); };
    constexpr int SHARED = APART ? 2 : 1; // tiles of K a step of two

    if (threadIdx.x == 0)
    {
        mbar_init(&b.q_full, 1);
        for (uint32_t s = 0; s < S::SLOTS; ++s)
            mbar_init(&b.full[s], 1), mbar_init(&b.empty[s], 1);
        for (int t = 0; t < 2; ++t)
        {
            for (int h = 0; h < 2; ++h)
                mbar_init(&b.s_full[t][h], 1), mbar_init(&b.p_ready[t][h], 4);
            mbar_init(&b.o_done[t], 1), mbar_init(&b.fin[t], 1);
        }
        b.give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == AT_MMA_WARP)
        at_tmem_alloc<S::COLUMNS>(&b.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, b.tmem, 0); // known to be uniform
    const int* p_index = p.q_side.count;
    wait_for_previous_kernel(p_index); // the sides' counts
    const AttnCells q(p.q_side, n, p.sq), kv(p.kv_side, n, p.sk);
    const int tiles = attn_tiles(kv.count, AT_TILE);
    int lo[2], steps[2]; // of either team: first tile of keys, steps of 64 keys
    for (int t = 0; t < 2; ++t)
    {
        const int part = APART ? 2 * split + t : split, first = APART ? 0 : i0 + t * AT_TILE;
        lo[t] = (int) ((long long) tiles * part / p.kv_splits);
        const int hi = (int) ((long long) tiles * (part + 1) / p.kv_splits);
        const int end = min(hi * AT_TILE, attn_limit(p, q, kv, min(first + AT_TILE, q.count) - 1)); // keys
        steps[t] = first < q.count ? max(0, end - lo[t] * AT_TILE + 63) / 64 : 0;
    }
    const int most = max(steps[0], steps[1]);
    bool ok = true;

    if (warp >= AT_MMA_WARP)
    {
        at_fewer_registers<S::OTHER_REGS>();
        if (warp == AT_TMA_WARP)
        {
            if (lane == 0 && most > 0)
            {
                const int own = APART ? 1 : 2; // query tiles
                mbar_expect_tx(&b.q_full, own * AtTile<D>::BYTES);
                for (int t = 0; t < own; ++t)
                    at_tma_tile<D>(base + S::Q_AT + t * AtTile<D>::BYTES, &maps.q, i0 + t * AT_TILE, head, (int) n,
                                   &b.q_full);
                AtRing r;
                const int loads = 2 * SHARED * ((most + 1) / 2);
                for (int u = 0; u < loads && ok; ++u)
                {
                    const int j = u / (2 * SHARED), t = u % SHARED;
                    const bool value = u % (2 * SHARED) >= SHARED;
                    if (r.lap > 0)
                        ok = mbar_wait_t<20>(&b.empty[r.slot], (r.lap - 1) & 1, give_up);
                    if (!ok)
                        break;
                    mbar_expect_tx(&b.full[r.slot], AtTile<D>::BYTES);
                    at_tma_tile<D>(base + S::RING_AT + r.slot * AtTile<D>::BYTES, value ? &maps.v : &maps.k,
                                   (lo[t] + j) * AT_TILE, kv_head, (int) n, &b.full[r.slot]);
                    r.next(S::SLOTS);
                }
                if (!ok || *give_up)
                {
                    int none = 0;
                    mbar_wait_t<20>(&b.q_full, 0, &none);
                    at_drain(b.full, S::SLOTS, r);
                }
            }
        }
        else if (warp == AT_MMA_WARP)
        {
            if (most > 0)
            {
                const uint32_t elected = at_elect();
                const int ksteps = (p.d + 15) / 16;
                const uint32_t width = (uint32_t) ksteps * 16;
                const auto tile_of = [&](uint32_t number) {
                    return base + S::RING_AT + number % S::SLOTS * AtTile<D>::BYTES;
                };
                const auto arrived = [&](uint32_t number) {
                    ok = ok && at_warp_wait(&b.full[number % S::SLOTS], number / S::SLOTS & 1, give_up);
                };
                const auto release = [&](uint32_t number) { at_commit(&b.empty[number % S::SLOTS], elected); };
                // every tile that was asked for is waited for, also by a team without work on it
                const auto keys_arrived = [&](int j) {
                    for (int t = 0; t < SHARED; ++t)
                        arrived(k_number(t, j));
                    tc_fence_after();
                };
                const auto scores = [&](int t, int u) {
                    at_scores<D, 64>(tmem + (t * S::PLACES + u % S::PLACES) * 64,
                                     base + S::Q_AT + (APART ? 0 : t * AtTile<D>::BYTES),
                                     tile_of(k_number(t, u >> 1)) + (u & 1) * AtTile<D>::HALF, ksteps, elected);
                    at_commit(&b.s_full[t][u % S::PLACES], elected);
                };
                ok = at_warp_wait(&b.q_full, 0, give_up);
                keys_arrived(0);
                // behind the last team's second half of a tile the slot is free
                const auto keys_done = [&](int u) {
                    if (ok && (u & 1) && u < most)
                        for (int t = 0; t < SHARED; ++t)
                            release(k_number(t, u >> 1));
                };
                for (int u = 0; u < S::PLACES; ++u)
                {
                    for (int t = 0; t < 2; ++t)
                        if (ok && u < steps[t])
                            scores(t, u);
                    keys_done(u);
                }
                for (int u = 0; u < most && ok; ++u)
                {
                    const int j = u >> 1, ahead = u + S::PLACES;
                    if ((u & 1) == 0)
                    {
                        for (int t = 0; t < SHARED; ++t)
                            arrived(v_number(t, j));
                        tc_fence_after();
                    }
                    bool have_k = ahead & 1;
                    // the teams in the order that they are ready in
                    uint32_t left = (u < steps[0] ? 1u : 0u) | (u < steps[1] ? 2u : 0u);
                    while (left && ok)
                    {
                        const int t = at_first_ready(&b.p_ready[0][u % S::PLACES], &b.p_ready[1][u % S::PLACES], left,
                                                     u / S::PLACES & 1, give_up);
                        ok = t >= 0;
                        if (!ok)
                            break;
                        left &= ~(1u << t);
                        tc_fence_after();
                        at_weigh<D>(tmem + S::O_AT + t * D, tmem + (t * S::PLACES + u % S::PLACES) * 64,
                                    tile_of(v_number(t, j)) + (u & 1) * AtTile<D>::HALF, width, u == 0, elected);
                        at_commit(&b.o_done[t], elected);
                        if (u + 1 == steps[t])
                            at_commit(&b.fin[t], elected);
                        if (ahead < steps[t])
                        {
                            if (!have_k)
                                keys_arrived(ahead >> 1);
                            have_k = true;
                            if (ok)
                                scores(t, ahead);
                        }
                    }
                    if (ok && (u & 1))
                        for (int t = 0; t < SHARED; ++t)
                            release(v_number(t, j));
                    keys_done(ahead);
                }
                if (!ok)
                {
                    // what was issued ends before the tensor memory is given back
                    int none = 0;
                    at_commit(&b.q_full, elected);
                    mbar_wait_t<20>(&b.q_full, 1, &none);
                }
            }
        }
    }
    else
    {
        at_more_registers<S::TEAM_REGS>();
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t) (warp & 3) << 21; // 32 lanes of tensor memory a warp
        const uint32_t o_at = tmem + lanes + S::O_AT + t * D;
        const int row0 = (APART ? 0 : i0 + t * AT_TILE) + (warp & 3) * 32, row = row0 + lane;
        const int i = row < q.count ? q.cell(row) : -1, limit = attn_limit(p, q, kv, row);
        const int part = APART ? 2 * split + t : split;
        const bool rows = row0 < q.count; // else no row of this warp is a cell: what its weights are reaches nobody
        float top = -INFINITY, sum = 0.f; // the base of the weights so far and their sum
        float mine = -INFINITY;           // the largest score of the step that comes next
        const auto score_at = [&](int u) { return tmem + lanes + (t * S::PLACES + u % S::PLACES) * 64; };
        const auto wait_scores = [&](int u) {
            ok = ok && at_warp_wait(&b.s_full[t][u % S::PLACES], u / S::PLACES & 1, give_up);
            tc_fence_after();
            return ok;
        };
        uint32_t see[2];  // which keys of the coming step this row may see
        bool cut = false; // whether some row of the warp may not see all of them
        const int open = max(0, attn_limit(p, q, kv, row0) - lo[t] * AT_TILE) / 64; // steps that all its rows see whole
        const auto mask = [&](int c, float x) { return see[c >> 5] >> (c & 31) & 1 ? x : -INFINITY; };
        // masks and maximum of a step's scores, which have arrived
        const auto look = [&](int u, float (&s)[64]) {
            cut = u >= open;
            if (cut)
            {
                const int j0 = lo[t] * AT_TILE + u * 64;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    see[w] = at_up_to(limit - 1 - j0, w);
#pragma unroll
                for (int c = 0; c < 64; ++c)
                    s[c] = mask(c, s[c]);
            }
            float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
            for (int c = 4; c < 60; c += 8)
            {
                m0 = at_max3(m0, s[c], s[c + 1]), m1 = at_max3(m1, s[c + 2], s[c + 3]);
                m2 = at_max3(m2, s[c + 4], s[c + 5]), m3 = at_max3(m3, s[c + 6], s[c + 7]);
            }
            m0 = at_max3(m0, s[60], s[61]), m1 = at_max3(m1, s[62], s[63]);
            mine = at_max3(fmaxf(m0, m1), m2, m3) * p.scale;
        };
        // The base of step u's weights; O follows where it grows.
        const auto renew = [&](int u) {
            const bool grown = mine > top + AF_GROWTH;
            if (!__any_sync(~0u, grown))
                return;
            const float shrink = grown ? at_exp2(top - mine) : 1.f;
            top = grown ? mine : top;
            sum *= shrink;
            if (u == 0)
                return;
            // O of the step before: with these scores' arrival all but that step have been added, and the next one waits
            // for this one's weights
            ok = at_warp_wait(&b.o_done[t], (u - 1) & 1, give_up);
            if (!ok)
                return;
            tc_fence_after();
            for (int c0 = 0; c0 < p.d; c0 += 32)
            {
                float o[32];
                at_tmem_ld32(o_at + c0, o);
                at_tmem_wait_ld();
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    o[c] *= shrink;
                at_tmem_st32(o_at + c0, reinterpret_cast<const uint32_t*>(o));
            }
        };
        uint64_t scale2, base2, l0, l1;
        const auto begin = [&] {
            const float base_of = top == -INFINITY ? 0.f : top;
            scale2 = at_pair(p.scale, p.scale), base2 = at_pair(-base_of, -base_of);
            l0 = l1 = 0;
        };
        // Weights of 16 scores, to the h-th eight columns.  With two blocks on an SM two of them do without ex2, whose
        // unit is what these warps wait for: 4 x 8 heads x 64^2 cells x 64 take 208 us, 219 with none, 208 with four, 226
        // with eight.  One block's warps have no issue slots left for it: 128 channels go from 611 us to 623.
        const auto weigh = [&](int u, int h, const float* s) {
            uint32_t w[8];
#pragma unroll
            for (int c = 0; c < 16; c += 4)
            {
                float e[4];
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                {
                    const uint64_t x = at_fma2(at_pair(s[c + k], s[c + k + 1]), scale2, base2);
                    if (S::BLOCKS == 2 && c + k == 14)
                        at_exp2_pair(x, e[k], e[k + 1]);
                    else
                    {
                        at_unpair(x, e[k], e[k + 1]);
                        e[k] = at_exp2(e[k]), e[k + 1] = at_exp2(e[k + 1]);
                    }
                }
                l0 = at_add2(l0, at_pair(e[0], e[1]));
                l1 = at_add2(l1, at_pair(e[2], e[3]));
                w[c / 2] = pack_bf16(e[0], e[1]);
                w[c / 2 + 1] = pack_bf16(e[2], e[3]);
            }
            tmem_st8(score_at(u) + 8 * h, w);
        };
        const auto hand_over = [&](int u) {
            float a, c;
            at_unpair(at_add2(l0, l1), a, c);
            sum += a + c;
            at_tmem_wait_st();
            at_warp_arrive(&b.p_ready[t][u % S::PLACES], lane);
        };
        const auto fetch = [&](int u, float (&s)[64]) {
            if (!wait_scores(u))
                return;
            at_tmem_ld32(score_at(u), s);
            at_tmem_ld32(score_at(u) + 32, s + 32);
            at_tmem_wait_ld();
            look(u, s);
        };
        if (steps[t] > 0 && rows)
        {
            if constexpr (S::BLOCKS == 1)
            {
                // Half way through step u the scores of the next one are fetched, which have been taken meanwhile.
                const auto step = [&](int u, float (&s)[64], float (&next)[64]) {
                    renew(u);
                    if (!ok)
                        return;
                    begin();
                    weigh(u, 0, s);
                    weigh(u, 1, s + 16);
                    if (u + 1 < steps[t])
                    {
                        if (!wait_scores(u + 1))
                            return;
                        at_tmem_ld32(score_at(u + 1), next);
                        at_tmem_ld32(score_at(u + 1) + 32, next + 32);
                    }
                    weigh(u, 2, s + 32);
                    weigh(u, 3, s + 48);
                    hand_over(u);
                    if (u + 1 < steps[t])
                    {
                        at_tmem_wait_ld();
                        look(u + 1, next);
                    }
                };
                float even[64], odd[64];
                fetch(0, even);
                for (int u = 0; u < steps[t] && ok; u += 2)
                {
                    step(u, even, odd);
                    if (u + 1 < steps[t] && ok)
                        step(u + 1, odd, even);
                }
            }
            else
            {
                // Half the registers: the scores are fetched once for their maximum and again, 16 at a time, for their
                // weights, which go over scores that have been fetched.
                for (int u = 0; u < steps[t] && ok; ++u)
                {
                    {
                        float s[64];
                        fetch(u, s);
                    }
                    if (ok)
                        renew(u);
                    if (!ok)
                        break;
                    begin();
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                    {
                        uint32_t raw[16];
                        float s[16];
                        tmem_ld16(score_at(u) + 16 * h, raw);
                        at_tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            s[c] = __uint_as_float(raw[c]);
                        if (cut)
                        {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                s[c] = mask(16 * h + c, s[c]);
                        }
                        weigh(u, h, s);
                    }
                    hand_over(u);
                }
            }
        }
        else
        {
            for (int u = 0; u < steps[t] && wait_scores(u); ++u)
                at_warp_arrive(&b.p_ready[t][u % S::PLACES], lane);
        }
        if (ok && steps[t] > 0)
            ok = at_warp_wait(&b.fin[t], 0, give_up); // o_done may be two steps away
        tc_fence_after();
        if (ok && rows)
        {
            const bool nothing = steps[t] == 0;
            const long long heads = (long long) p.n * p.q_heads;
            if (p.kv_splits > 1)
            {
                if (i >= 0)
                {
                    float* ml = p.part_ml + (2 * heads * part + nh) * p.sq + i;
                    ml[0] = top;
                    ml[heads * p.sq] = sum;
                }
                at_store(p.o, p.part_o + part * heads * p.d * p.sq, nh, n, head, p.d, i, p.sq, 1.f, false, nothing, o_at,
                         0, D);
            }
            else
            {
                const bool none = sum == 0.f;
                at_store(p.o, nullptr, nh, n, head, p.d, i, p.sq, 1.f / sum, none, nothing, o_at, 0, D);
                if (i >= 0)
                    p.lse[nh * p.sq + i] = none ? -INFINITY : (top + log2f(sum)) / ATTN_LOG2E;
            }
        }
    }
    at_finish<S::COLUMNS>(ok, warp, lane, tmem);
}

template <int D, bool APART>
int32_t af_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream)
{
    const long long blocks = (long long) p.n * p.q_heads
                             * (APART ? p.kv_splits / 2 : (long long) attn_tiles(p.sq, 2 * AT_TILE) * p.kv_splits);
    DCB_REQUIRE(blocks < (1ll << 31), "too many tiles");
    if (int32_t e = allow_dynamic_smem((const void*) attn_tc_fwd_kernel<D, APART>, AfShape<D, APART>::SMEM))
        return e;
    DCB_CUDA_TRY(launch_overlapped(attn_tc_fwd_kernel<D, APART>, dim3((unsigned) blocks), AT_THREADS, AfShape<D, APART>::SMEM,
                                   stream, p, maps));
    return DCB_OK;
}

} // namespace

int32_t attn_tc_fwd_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream)
{
    if (attn_tc_apart(p))
        return af_launch<64, true>(p, maps, stream);
    return p.d <= 64 ? af_launch<64, false>(p, maps, stream) : af_launch<128, false>(p, maps, stream);
}

int32_t attn_tc_fwd_status(bool* gave_up)
{
    return at_read_status(gave_up);
}

} // namespace dcb
