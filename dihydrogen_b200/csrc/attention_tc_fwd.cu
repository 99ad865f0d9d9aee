// Attention forward on the tensor cores.
//
// A block has two tiles of 128 query cells of one head, each with a team of 128 threads, one row a
// thread, and walks over tiles of 128 keys.  While one team turns its scores into weights the tensor
// cores work for the other: S = Q K' into 128 columns of tensor memory, then, the weights written
// back as bf16 over the scores, O += P V.  A row's weights are powers of two about a maximum that
// is renewed only when it has grown by more than 2^8 since; then the thread scales its row of O.
// (The sums are exact about any base that keeps them in range.)
#include "attention_tc.cuh"

namespace dcb
{

namespace
{

constexpr float AF_GROWTH = 8.f;

template <int D>
struct AfShape
{
    static constexpr uint32_t SLOTS = D == 128 ? 5 : 8; // of K and V tiles in turn
    static constexpr uint32_t Q_AT = 0;
    static constexpr uint32_t RING_AT = 2 * AtTile<D>::BYTES;
    static constexpr uint32_t BARS_AT = RING_AT + SLOTS * AtTile<D>::BYTES;
    static constexpr uint32_t SMEM = BARS_AT + 256;
};

struct AfBars
{
    uint64_t q_full, full[8], empty[8], s_full[2], p_ready[2], o_full[2];
    uint32_t tmem;
    int give_up;
};
static_assert(sizeof(AfBars) <= 256, "the barriers' room");

template <int D>
__global__ void __launch_bounds__(AT_THREADS, 1)
    attn_tc_fwd_kernel(const __grid_constant__ AttnProblem p, const __grid_constant__ AtMaps maps,
                       const __grid_constant__ AtExtra ex)
{
    using S = AfShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    AfBars& b = *reinterpret_cast<AfBars*>(smem + S::BARS_AT);
    const int warp = __shfl_sync(~0u, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    volatile int* give_up = &b.give_up;
    if (at_misplaced(base, ex.status))
        return;

    long long at = blockIdx.x;
    const int blocks_q = attn_tiles(p.sq, 2 * AT_TILE);
    const int block_q = blocks_q - 1 - (int) (at % blocks_q); // causal: the longest walks first
    at /= blocks_q;
    const int split = (int) (at % p.kv_splits);
    const long long nh = at / p.kv_splits, n = nh / p.q_heads;
    const int head = (int) (nh - n * p.q_heads), kv_head = head / p.group;
    const int i0 = block_q * 2 * AT_TILE;
    const int tiles = attn_tiles(p.sk, AT_TILE);
    const int lo = (int) ((long long) tiles * split / p.kv_splits);
    const int hi = (int) ((long long) tiles * (split + 1) / p.kv_splits);
    int steps[2]; // of either team
    for (int t = 0; t < 2; ++t)
    {
        const int first = i0 + t * AT_TILE;
        int end = hi;
        if (p.causal)
            end = (int) min((long long) hi, max(0ll, (long long) first + AT_TILE - 1 + p.offset + AT_TILE) / AT_TILE);
        steps[t] = first < p.sq ? max(0, end - lo) : 0;
    }
    const int most = max(steps[0], steps[1]);

    if (threadIdx.x == 0)
    {
        mbar_init(&b.q_full, 1);
        for (uint32_t s = 0; s < S::SLOTS; ++s)
            mbar_init(&b.full[s], 1), mbar_init(&b.empty[s], 1);
        for (int t = 0; t < 2; ++t)
            mbar_init(&b.s_full[t], 1), mbar_init(&b.p_ready[t], 4), mbar_init(&b.o_full[t], 1);
        b.give_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == AT_MMA_WARP)
        at_tmem_alloc(&b.tmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, b.tmem, 0); // known to be uniform
    const uint32_t* bits = ex.kv_bits ? ex.kv_bits + n * ex.words : nullptr;
    wait_for_previous_kernel(bits);
    bool ok = true;

    if (warp >= AT_MMA_WARP)
    {
        at_other_registers();
        if (warp == AT_TMA_WARP)
        {
            if (lane == 0 && most > 0)
            {
                mbar_expect_tx(&b.q_full, 2 * AtTile<D>::BYTES);
                for (int t = 0; t < 2; ++t)
                    at_tma_tile<D>(base + S::Q_AT + t * AtTile<D>::BYTES, &maps.q, i0 + t * AT_TILE, head, (int) n,
                                   &b.q_full);
                AtRing r;
                for (int u = 0; u < 2 * most && ok; ++u)
                {
                    if (r.lap > 0)
                        ok = mbar_wait_t<20>(&b.empty[r.slot], (r.lap - 1) & 1, give_up);
                    if (!ok)
                        break;
                    mbar_expect_tx(&b.full[r.slot], AtTile<D>::BYTES);
                    at_tma_tile<D>(base + S::RING_AT + r.slot * AtTile<D>::BYTES, u & 1 ? &maps.v : &maps.k,
                                   (lo + (u >> 1)) * AT_TILE, kv_head, (int) n, &b.full[r.slot]);
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
                const auto tile_of = [&](uint32_t slot) { return base + S::RING_AT + slot * AtTile<D>::BYTES; };
                AtRing r; // the tile after the last one that was waited for
                ok = at_warp_wait(&b.q_full, 0, give_up) && at_warp_wait(&b.full[r.slot], r.lap & 1, give_up);
                tc_fence_after();
                uint32_t k_slot = r.slot;
                r.next(S::SLOTS);
                for (int t = 0; t < 2 && ok; ++t)
                    if (steps[t] > 0)
                    {
                        at_scores<D>(tmem + t * AT_TILE, base + S::Q_AT + t * AtTile<D>::BYTES, tile_of(k_slot), ksteps,
                                     elected);
                        at_commit(&b.s_full[t], elected);
                    }
                if (ok)
                    at_commit(&b.empty[k_slot], elected);
                for (int j = 0; j < most && ok; ++j)
                {
                    const uint32_t v_slot = r.slot;
                    ok = at_warp_wait(&b.full[r.slot], r.lap & 1, give_up);
                    r.next(S::SLOTS);
                    bool have_k = false;
                    for (int t = 0; t < 2 && ok; ++t)
                    {
                        if (j < steps[t])
                        {
                            ok = at_warp_wait(&b.p_ready[t], j & 1, give_up);
                            if (!ok)
                                break;
                            tc_fence_after();
                            at_weigh<D>(tmem + 2 * AT_TILE + t * D, tmem + t * AT_TILE, 32, tile_of(v_slot), width, j == 0,
                                    elected);
                            if (j + 1 == steps[t])
                                at_commit(&b.o_full[t], elected);
                        }
                        if (t == 1)
                            at_commit(&b.empty[v_slot], elected);
                        if (j + 1 < steps[t])
                        {
                            if (!have_k)
                            {
                                ok = at_warp_wait(&b.full[r.slot], r.lap & 1, give_up);
                                if (!ok)
                                    break;
                                tc_fence_after();
                                have_k = true;
                            }
                            at_scores<D>(tmem + t * AT_TILE, base + S::Q_AT + t * AtTile<D>::BYTES, tile_of(r.slot), ksteps, elected);
                            at_commit(&b.s_full[t], elected);
                        }
                    }
                    if (ok && j + 1 < most)
                    {
                        at_commit(&b.empty[r.slot], elected);
                        r.next(S::SLOTS);
                    }
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
        at_team_registers();
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t) (warp & 3) << 21; // 32 lanes of tensor memory a warp
        const uint32_t s_at = tmem + lanes + t * AT_TILE, o_at = tmem + lanes + 2 * AT_TILE + t * D;
        const int i = i0 + t * AT_TILE + (threadIdx.x & 127);
        float top = -INFINITY, sum = 0.f; // the base of the weights so far and their sum
        for (int j = 0; j < steps[t]; ++j)
        {
            const int j0 = (lo + j) * AT_TILE;
            ok = at_warp_wait(&b.s_full[t], j & 1, give_up);
            if (!ok)
                break;
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                at_tmem_ld32(s_at + 32 * c, s + 32 * c);
            at_tmem_wait_ld();
            uint32_t see[4];
            bool all = true;
#pragma unroll
            for (int w = 0; w < 4; ++w)
            {
                see[w] = at_there(p, bits, j0, w);
                if (p.causal)
                    see[w] &= at_up_to(i + p.offset - j0, w);
                all = all && see[w] == ~0u;
            }
            if (__any_sync(~0u, !all))
            {
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    s[c] = see[c >> 5] >> (c & 31) & 1 ? s[c] : -INFINITY;
            }
            float m0 = s[0], m1 = s[1], m2 = s[2], m3 = s[3];
#pragma unroll
            for (int c = 4; c < 124; c += 8)
            {
                m0 = at_max3(m0, s[c], s[c + 1]), m1 = at_max3(m1, s[c + 2], s[c + 3]);
                m2 = at_max3(m2, s[c + 4], s[c + 5]), m3 = at_max3(m3, s[c + 6], s[c + 7]);
            }
            m0 = at_max3(m0, s[124], s[125]), m1 = at_max3(m1, s[126], s[127]);
            const float mine = at_max3(fmaxf(m0, m1), m2, m3) * p.scale;
            const bool grown = mine > top + AF_GROWTH;
            if (__any_sync(~0u, grown))
            {
                const float shrink = grown ? at_exp2(top - mine) : 1.f;
                top = grown ? mine : top;
                sum *= shrink;
                if (j > 0)
                {
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
                }
            }
            const float base_of = top == -INFINITY ? 0.f : top;
            float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half)
            {
                uint32_t w[32];
#pragma unroll
                for (int c = 0; c < 64; c += 4)
                {
                    const float* x = s + 64 * half + c;
                    const float e0 = at_exp2(fmaf(x[0], p.scale, -base_of)), e1 = at_exp2(fmaf(x[1], p.scale, -base_of));
                    const float e2 = at_exp2(fmaf(x[2], p.scale, -base_of)), e3 = at_exp2(fmaf(x[3], p.scale, -base_of));
                    l0 += e0, l1 += e1, l2 += e2, l3 += e3;
                    w[c / 2] = pack_bf16(e0, e1);
                    w[c / 2 + 1] = pack_bf16(e2, e3);
                }
                at_tmem_st32(s_at + 32 * half, w);
            }
            sum += (l0 + l1) + (l2 + l3);
            at_tmem_wait_st();
            at_warp_arrive(&b.p_ready[t], lane);
        }
        if (ok && steps[t] > 0)
            ok = at_warp_wait(&b.o_full[t], 0, give_up);
        tc_fence_after();
        if (ok)
        {
            const bool nothing = steps[t] == 0;
            if (i0 + t * AT_TILE < p.sq)
            {
                const long long heads = (long long) p.n * p.q_heads;
                if (p.kv_splits > 1)
                {
                    if (i < p.sq)
                    {
                        float* ml = p.part_ml + (2 * heads * split + nh) * p.sq + i;
                        ml[0] = top;
                        ml[heads * p.sq] = sum;
                    }
                    at_store(p.o, p.part_o + split * heads * p.d * p.sq, nh, n, head, p.d, i, p.sq, 1.f, false, nothing,
                             o_at, 0, D);
                }
                else
                {
                    const bool none = sum == 0.f || (p.q_mask && i < p.sq && !p.q_mask[n * p.sq + i]);
                    at_store(p.o, nullptr, nh, n, head, p.d, i, p.sq, 1.f / sum, none, nothing, o_at, 0, D);
                    if (i < p.sq)
                        p.lse[nh * p.sq + i] = none ? -INFINITY : (top + log2f(sum)) / ATTN_LOG2E;
                }
            }
        }
    }
    at_finish(ok, ex.status, warp, lane, tmem);
}

template <int D>
int32_t af_launch(const AttnProblem& p, const AtMaps& maps, const AtExtra& ex, cudaStream_t stream)
{
    const long long blocks = (long long) p.n * p.q_heads * attn_tiles(p.sq, 2 * AT_TILE) * p.kv_splits;
    DCB_REQUIRE(blocks < (1ll << 31), "too many tiles");
    if (int32_t e = allow_dynamic_smem((const void*) attn_tc_fwd_kernel<D>, AfShape<D>::SMEM))
        return e;
    DCB_CUDA_TRY(launch_overlapped(attn_tc_fwd_kernel<D>, dim3((unsigned) blocks), AT_THREADS, AfShape<D>::SMEM, stream,
                                   p, maps, ex));
    return DCB_OK;
}

} // namespace

int32_t attn_tc_fwd_launch(const AttnProblem& p, const AtMaps& maps, const AtExtra& ex, cudaStream_t stream)
{
    return p.d <= 64 ? af_launch<64>(p, maps, ex, stream) : af_launch<128>(p, maps, ex, stream);
}

} // namespace dcb
