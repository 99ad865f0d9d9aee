// Attention of a few queries: a pass over the keys and values, bound by memory.
//
// A block has one query of one head and a part of the keys; a warp has 8 or 16 channels, a lane 8 keys of the tile: 16
// bytes of neighbours at a time, or keys 32 apart through their indices where rows are off alignment or a mask picks
// them.  The warps exchange their channels' shares of the scores through shared memory, before which the values are on
// their way; every lane then weighs its keys about a maximum of its own and adds up its channels of the values: the
// lanes' sums meet at the block's end.  Parts are joined by a kernel of their own.  Weights stay fp32.
//
// 2 x 8 heads x 64, a query each, parts' join included: bf16, 32^3 keys 36 us (134 MB: 3.7 TB/s; start, the
// parts' last tiles and the join are 12 of it), 32 x 64 x 64 keys 100 us (5.4 TB/s); fp32, 20 x 20 x 65 keys 43 us (213 MB:
// 5 TB/s).
#include "attention.cuh"

namespace dcb
{
namespace
{

constexpr int ATH_KEYS = 8; // of a lane, in a tile
constexpr float ATH_GROWTH = 8.f; // a lane's base is renewed where a score is more than 2^8 above it

template <class T, bool GATHER>
struct AthKeys
{
    static constexpr int WIDE = GATHER ? 1 : 16 / sizeof(T), LOADS = ATH_KEYS / WIDE;
    int first, at[LOADS]; // the lane's first key, cells
    __device__ __forceinline__ AthKeys(const AttnCells& kv, int j0, int lane, int end)
    {
        first = j0 + lane * WIDE;
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
        {
            const int j = key(l * WIDE) < end ? key(l * WIDE) : 0;
            at[l] = GATHER ? kv.cell(j) : j;
        }
    }
    __device__ __forceinline__ int key(int e) const { return first + (e / WIDE) * 32 * WIDE + e % WIDE; }
    struct Values
    {
        RawElems<T, WIDE> r[LOADS];
        __device__ __forceinline__ float get(int e) const { return r[e / WIDE].get(e % WIDE); }
    };
    __device__ __forceinline__ void load(Values& v, const T* row) const
    {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
            v.r[l].load(row + at[l]);
    }
};

template <class T, int WARPS, int CHANNELS, bool GATHER>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) attn_thin_fwd_kernel(const __grid_constant__ AttnProblem p)
{
    typedef AthKeys<T, GATHER> Keys;
    constexpr int V = ATH_KEYS;
    __shared__ float query[WARPS * CHANNELS];
    __shared__ float shares[WARPS][V][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = warp * CHANNELS;
    // the queries that read a key head come one after the other: what the first reads is in L2 for the rest
    long long at = blockIdx.x;
    const int row = (int) (at % p.sq);
    at /= p.sq;
    const int g = (int) (at % p.group);
    at /= p.group;
    const int split = (int) (at % p.kv_splits);
    at /= p.kv_splits;
    const long long n = at / p.kv_heads;
    const int kv_head = (int) (at - n * p.kv_heads), head = kv_head * p.group + g;
    const long long nh = n * p.q_heads + head;
    const float* lse = p.lse;
    wait_for_previous_kernel(lse);
    dependents_may_start();
    const AttnCells q(p.q_side, n, p.sq), kv(p.kv_side, n, p.sk);
    if (row >= q.count)
        return;
    const int i = q.cell(row), limit = attn_limit(p, q, kv, row);
    // parts are whole units of 64 keys (a line of 128 bytes of bf16): the last tile of a part may be cut short
    const int units = attn_tiles(limit, 64);
    const int lo = 64 * (int) ((long long) units * split / p.kv_splits);
    const int hi = min(64 * (int) ((long long) units * (split + 1) / p.kv_splits), limit);
    {
        const int c = threadIdx.x;
        if (c < WARPS * CHANNELS)
        {
            float v[1] = {0.f};
            if (c < p.d)
                load_elems<1>(static_cast<const T*>(p.q.p) + n * p.q.sn + ((long long) head * p.d + c) * p.q.sc + i, v);
            query[c] = v[0] * p.scale;
        }
    }
    __syncthreads();

    const int channels = min(CHANNELS, p.d - c0); // may be negative: the last channel is fetched in place of those past it
    const T* keys = static_cast<const T*>(p.k.p) + n * p.k.sn + (long long) kv_head * p.d * p.k.sc;
    const T* values = static_cast<const T*>(p.v.p) + n * p.v.sn + (long long) kv_head * p.d * p.v.sc;
    float top = -INFINITY, sum = 0.f, acc[CHANNELS];
#pragma unroll
    for (int c = 0; c < CHANNELS; ++c)
        acc[c] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 32 * V)
    {
        const Keys mine(kv, j0, lane, hi);
        typename Keys::Values k[CHANNELS], v[CHANNELS];
#pragma unroll
        for (int c = 0; c < CHANNELS; ++c)
            mine.load(k[c], keys + min(c0 + c, p.d - 1) * p.k.sc);
        float s[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
            s[e] = 0.f;
#pragma unroll
        for (int c = 0; c < CHANNELS; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e)
                s[e] = c < channels ? fmaf(query[c0 + c], k[c].get(e), s[e]) : s[e];
        if (WARPS > 1)
        {
#pragma unroll
            for (int e = 0; e < V; ++e)
                shares[warp][e][lane] = s[e];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                s[e] = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w)
                    s[e] += shares[w][e][lane];
            }
        }
#pragma unroll
        for (int c = 0; c < CHANNELS; ++c)
            mine.load(v[c], values + min(c0 + c, p.d - 1) * p.v.sc);
        __syncthreads(); // the next tile's shares
        float most = -INFINITY;
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            s[e] = mine.key(e) < hi ? s[e] : -INFINITY;
            most = fmaxf(most, s[e]);
        }
        if (most > top + ATH_GROWTH)
        {
            const float shrink = exp2f(top - most);
            top = most;
            sum *= shrink;
#pragma unroll
            for (int c = 0; c < CHANNELS; ++c)
                acc[c] *= shrink;
        }
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            s[e] = exp2f(s[e] - base);
            sum += s[e];
        }
#pragma unroll
        for (int c = 0; c < CHANNELS; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e)
                acc[c] = fmaf(s[e], v[c].get(e), acc[c]);
    }

    // one base for the lanes, whose keys are the same in every warp
    float m = top;
#pragma unroll
    for (int h = 16; h >= 1; h /= 2)
        m = fmaxf(m, __shfl_xor_sync(~0u, m, h));
    const float f = top == -INFINITY ? 0.f : exp2f(top - m);
    sum *= f;
#pragma unroll
    for (int h = 16; h >= 1; h /= 2)
        sum += __shfl_xor_sync(~0u, sum, h);
#pragma unroll
    for (int c = 0; c < CHANNELS; ++c)
        acc[c] *= f;
    const float o = lane_sums<CHANNELS>(acc, lane);
    const long long heads = (long long) p.n * p.q_heads;
    const int c = c0 + lane;
    if (lane < channels)
    {
        if (p.kv_splits > 1)
            p.part_o[((split * heads + nh) * p.d + c) * p.sq + i] = o;
        else
        {
            const float v[1] = {sum == 0.f ? 0.f : o / sum};
            store_elems<1>(static_cast<T*>(p.o.p) + n * p.o.sn + ((long long) head * p.d + c) * p.o.sc + i, v);
        }
    }
    if (threadIdx.x == 0)
    {
        if (p.kv_splits > 1)
        {
            p.part_ml[(2 * heads * split + nh) * p.sq + i] = m;
            p.part_ml[(2 * heads * split + heads + nh) * p.sq + i] = sum;
        }
        else
            p.lse[nh * p.sq + i] = sum == 0.f ? -INFINITY : (m + log2f(sum)) / ATTN_LOG2E;
    }
}

// Channels of a warp where the keys are neighbours.  2 x 8 heads x 64, a query each: bf16 with 32^3 keys takes 31 us
// with 16 and 36 with 8, fp32 with 20 x 20 x 65 keys 65 us and 43.  Through indices it is 8: 16 spill.
template <class T>
constexpr int ath_channels()
{
    return sizeof(T) == 2 ? 16 : 8;
}

template <class T>
int32_t ath_fwd(const AttnProblem& p, cudaStream_t stream)
{
    constexpr int V = 16 / sizeof(T);
    const long long blocks = (long long) p.n * p.q_heads * p.sq * p.kv_splits;
    DCB_REQUIRE(blocks < (1ll << 31), "too many queries");
    const auto aligned = [&](const AttnTensor& t) {
        return reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.sc % V == 0 && (p.n == 1 || t.sn % V == 0);
    };
    // accesses of V cells, none of which reaches behind a row
    const bool gather = p.kv_mask || p.sk % V != 0 || !aligned(p.k) || !aligned(p.v);
    const auto go = [&](auto kernel, int warps) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(kernel, dim3((unsigned) blocks), 32 * warps, 0, stream, p));
        return DCB_OK;
    };
    const auto sized = [&](auto w) -> int32_t {
        constexpr int WARPS = decltype(w)::value;
        if (gather)
            return go(attn_thin_fwd_kernel<T, WARPS, 8, true>, WARPS);
        constexpr int CHANNELS = ath_channels<T>();
        return go(attn_thin_fwd_kernel<T, WARPS * 8 / CHANNELS, CHANNELS, false>, WARPS * 8 / CHANNELS);
    };
    if (p.d <= 32)
        return sized(std::integral_constant<int, 4>());
    if (p.d <= 64)
        return sized(std::integral_constant<int, 8>());
    return sized(std::integral_constant<int, 16>());
}

} // namespace

bool attn_thin(const AttnProblem& p, int32_t dtype)
{
    return p.sq <= (dtype == DCB_BF16 ? ATTN_THIN_BF16 : ATTN_THIN_F32);
}

void attn_thin_splits(AttnProblem* p, int32_t dtype)
{
    // the blocks that run at a time, 16 warps an SM; a part has a tile at least
    const int channels = dtype == DCB_BF16 && !p->kv_mask && p->sk % 8 == 0 ? ath_channels<bf16>() : 8;
    const int warps = (p->d <= 32 ? 32 : p->d <= 64 ? 64 : 128) / channels;
    p->kv_splits = attn_splits((long long) p->n * p->q_heads * p->sq, attn_tiles(p->sk, 32 * ATH_KEYS),
                               (16ll / warps) * num_sms());
    p->q_splits = 1;
}

int32_t attn_thin_fwd(const AttnProblem& p, int32_t dtype, cudaStream_t stream)
{
    return dtype == DCB_BF16 ? ath_fwd<bf16>(p, stream) : ath_fwd<float>(p, stream);
}

} // namespace dcb
