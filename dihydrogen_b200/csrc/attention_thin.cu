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
// Keys of a part, at most, forward: a lane adds up a 32nd of them one after the other, and after 2^15 terms of like size
// such a sum was off by 2.6e-4 (2^10: 4e-6 at most).  More than so many parts would be a long sum themselves.  40 x 8
// queries on 4 key heads of 64, 2^18 keys, fp32: 4.1 ms, in whole walks 7.0.
constexpr int ATH_PART_KEYS = 1 << 15, ATH_MOST_PARTS = 4096;
constexpr float ATH_GROWTH = 8.f; // a lane's base is renewed where a score is more than 2^8 above it

template <class T, int KEYS, bool GATHER>
struct AthKeys
{
    static constexpr int WIDE = GATHER ? 1 : 16 / sizeof(T), LOADS = KEYS / WIDE;
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
    // Values of keys from `end` on are 0: a weight of 0 times an infinity that was fetched in their place would not be.
    // Where a lane's keys are one access its condition costs nothing (2 x 8 heads x 64 over 32^3 bf16 keys: 38.8 us, 40.2
    // with a look behind the loads); with eight of them it does (31 x 33 x 31 keys: 98 us and 75).
    __device__ __forceinline__ void load_until(Values& v, const T* row, int end) const
    {
        if (LOADS > 1 || first < end)
            load(v, row);
        else
            v.r[0].clear();
    }
    __device__ __forceinline__ void clear_behind(Values& v, int end) const
    {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
            if (key(l * WIDE) >= end)
                v.r[l].clear();
    }
    // keys up to `end`, which WIDE divides or which is the last
    __device__ __forceinline__ void store(T* row, const float (&v)[KEYS], int end) const
    {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
            if (key(l * WIDE) < end)
            {
                float x[WIDE];
#pragma unroll
                for (int e = 0; e < WIDE; ++e)
                    x[e] = v[l * WIDE + e];
                store_elems<WIDE>(row + at[l], x);
            }
    }
};

template <class T, int WARPS, int CHANNELS, bool GATHER>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) attn_thin_fwd_kernel(const __grid_constant__ AttnProblem p)
{
    typedef AthKeys<T, ATH_KEYS, GATHER> Keys;
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
            mine.load_until(v[c], values + min(c0 + c, p.d - 1) * p.v.sc, hi);
        __syncthreads(); // the next tile's shares
        if (Keys::LOADS > 1 && j0 + 32 * V > hi)
#pragma unroll
            for (int c = 0; c < CHANNELS; ++c)
                mine.clear_behind(v[c], hi);
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

constexpr int ATH_ROWS = 16;     // queries, of all heads that read a key head, of the backward kernel at most
constexpr int ATH_BWD_KEYS = 4; // of a lane, in a tile of that

// Backward, fp32: a block has a part of a key head's keys and every query that reads them; a warp has 8 channels, a lane
// 4 keys.  Keys and values are read once, dk and dv have one owner and are written once; dq is added up over the block's
// keys in shared memory, and over the parts by a kernel of its own.  Scores and dP come of the warps' shares as forward.
// With a query bound by memory (2 x 8 heads of 64, 20 x 20 x 65 keys 97 us: 4.4 TB/s), with more by the exchanges.
template <int WARPS, bool GATHER>
__global__ void __launch_bounds__(32 * WARPS, 16 / WARPS) attn_thin_bwd_kernel(const __grid_constant__ AttnProblem p)
{
    constexpr int C = 8, V = ATH_BWD_KEYS;
    typedef AthKeys<float, V, GATHER> Keys;
    __shared__ float qs[ATH_ROWS][WARPS * C], gs[ATH_ROWS][WARPS * C], dqs[ATH_ROWS][WARPS * C];
    __shared__ float shares[WARPS][2 * V][32];
    __shared__ float lses[ATH_ROWS], deltas[ATH_ROWS];
    __shared__ int limits[ATH_ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = warp * C;
    long long at = blockIdx.x;
    const int split = (int) (at % p.kv_splits);
    at /= p.kv_splits;
    const long long n = at / p.kv_heads;
    const int kv_head = (int) (at - n * p.kv_heads);
    const float* stats = p.stats;
    wait_for_previous_kernel(stats);
    dependents_may_start();
    const AttnCells q(p.q_side, n, p.sq), kv(p.kv_side, n, p.sk);
    const long long heads = (long long) p.n * p.q_heads, nh0 = n * p.q_heads + kv_head * p.group;
    const int rows = p.group * q.count;
    for (int r = warp; r < rows; r += WARPS)
    {
        const int g = r / q.count, i = r - g * q.count, cell = q.cell(i);
        const long long head = kv_head * p.group + g;
        for (int c = lane; c < WARPS * C; c += 32)
        {
            const bool in = c < p.d;
            const long long row = head * p.d + c;
            qs[r][c] = in ? static_cast<const float*>(p.q.p)[n * p.q.sn + row * p.q.sc + cell] * p.scale : 0.f;
            gs[r][c] = in ? static_cast<const float*>(p.d_o.p)[n * p.d_o.sn + row * p.d_o.sc + cell] : 0.f;
            dqs[r][c] = 0.f;
        }
        if (lane == 0)
        {
            lses[r] = stats[(nh0 + g) * p.stats_pitch + i];
            deltas[r] = stats[(heads + nh0 + g) * p.stats_pitch + i];
            limits[r] = attn_limit(p, q, kv, i);
        }
    }
    __syncthreads();

    const int units = attn_tiles(kv.count, 32); // a line of 128 bytes
    const int lo = 32 * (int) ((long long) units * split / p.kv_splits);
    const int hi = min(32 * (int) ((long long) units * (split + 1) / p.kv_splits), kv.count);
    const long long first = (long long) kv_head * p.d;
    const float* keys = static_cast<const float*>(p.k.p) + n * p.k.sn + first * p.k.sc;
    const float* values = static_cast<const float*>(p.v.p) + n * p.v.sn + first * p.v.sc;
    float* dk_of = static_cast<float*>(p.dk.p) + n * p.dk.sn + first * p.dk.sc;
    float* dv_of = static_cast<float*>(p.dv.p) + n * p.dv.sn + first * p.dv.sc;
    for (int j0 = lo; j0 < hi; j0 += 32 * V)
    {
        const Keys mine(kv, j0, lane, hi);
        typename Keys::Values k[C], v[C];
#pragma unroll
        for (int c = 0; c < C; ++c)
        {
            mine.load(k[c], keys + min(c0 + c, p.d - 1) * p.k.sc);
            mine.load(v[c], values + min(c0 + c, p.d - 1) * p.v.sc);
        }
        float dk[C][V], dv[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e)
                dk[c][e] = dv[c][e] = 0.f;
        for (int r = 0; r < rows; ++r)
        {
            float s[V], dp[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
                s[e] = dp[e] = 0.f;
#pragma unroll
            for (int c = 0; c < C; ++c)
                if (c0 + c < p.d)
#pragma unroll
                    for (int e = 0; e < V; ++e)
                    {
                        s[e] = fmaf(qs[r][c0 + c], k[c].get(e), s[e]);
                        dp[e] = fmaf(gs[r][c0 + c], v[c].get(e), dp[e]);
                    }
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                shares[warp][e][lane] = s[e];
                shares[warp][V + e][lane] = dp[e];
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                s[e] = dp[e] = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w)
                {
                    s[e] += shares[w][e][lane];
                    dp[e] += shares[w][V + e][lane];
                }
                const bool seen = mine.key(e) < min(hi, limits[r]);
                s[e] = seen ? exp2f(s[e] - lses[r]) : 0.f;
                dp[e] = seen ? s[e] * (dp[e] - deltas[r]) : 0.f;
            }
            __syncthreads(); // the next row's shares
            float dq[C];
#pragma unroll
            for (int c = 0; c < C; ++c)
            {
                dq[c] = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e)
                {
                    dv[c][e] = fmaf(s[e], gs[r][c0 + c], dv[c][e]);
                    dk[c][e] = fmaf(dp[e], qs[r][c0 + c], dk[c][e]);
                    dq[c] = fmaf(dp[e], k[c].get(e), dq[c]);
                }
            }
            const float sum = lane_sums<C>(dq, lane);
            if (lane < C)
                dqs[r][c0 + lane] += sum; // of this warp's channels
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
            if (c0 + c < p.d)
            {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    dk[c][e] *= 1.f / ATTN_LOG2E; // q was multiplied with scale log2(e)
                mine.store(dk_of + (c0 + c) * p.dk.sc, dk[c], hi);
                mine.store(dv_of + (c0 + c) * p.dv.sc, dv[c], hi);
            }
    }
    const float factor = p.scale / ATTN_LOG2E;
    __syncwarp();
    for (int r = 0; r < rows; ++r)
        if (lane < C && c0 + lane < p.d)
        {
            const int g = r / q.count, cell = q.cell(r - g * q.count), c = c0 + lane;
            const float x = dqs[r][c] * factor;
            if (p.kv_splits > 1)
                p.part_dq[(((long long) split * heads + nh0 + g) * p.d + c) * p.sq + cell] = x;
            else
                static_cast<float*>(p.dq.p)[n * p.dq.sn + ((long long) (kv_head * p.group + g) * p.d + c) * p.dq.sc + cell]
                    = x;
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
    // the blocks that run at a time, 16 warps an SM; a part has a tile at least, ATH_PART_KEYS at most
    const int channels = dtype == DCB_BF16 && !p->kv_mask && p->sk % 8 == 0 ? ath_channels<bf16>() : 8;
    const int warps = (p->d <= 32 ? 32 : p->d <= 64 ? 64 : 128) / channels;
    p->kv_splits = std::max(attn_splits((long long) p->n * p->q_heads * p->sq, attn_tiles(p->sk, 32 * ATH_KEYS),
                                        (16ll / warps) * num_sms()),
                            std::min(attn_tiles(p->sk, ATH_PART_KEYS), ATH_MOST_PARTS));
    p->q_splits = 1;
}

// fp32, against the kernels of attention_simt.cu (dk, dv and dq, their join): 2 x 8 heads of 64, 20 x 20 x 65 keys, a query
// 97 us and 1120, four 184, sixteen 580; 2 x 4 heads of 128, 64^2 keys, sixteen 140 us and 190; 2 heads of 64, 256 keys,
// eight 22 us and 33, sixteen 42.
bool attn_thin_backward(const AttnProblem& p, int32_t dtype)
{
    return dtype == DCB_F32 && (long long) p.sq * p.group <= (p.sk >= 4096 ? ATH_ROWS : ATH_ROWS / 2);
}

void attn_thin_bwd_splits(AttnProblem* p)
{
    const int warps = (p->d <= 32 ? 32 : p->d <= 64 ? 64 : 128) / 8;
    p->kv_splits = attn_splits((long long) p->n * p->kv_heads, attn_tiles(p->sk, 32 * ATH_BWD_KEYS),
                               (16ll / warps) * num_sms());
    p->q_splits = 1;
}

int32_t attn_thin_bwd(const AttnProblem& p, cudaStream_t stream)
{
    const long long blocks = (long long) p.n * p.kv_heads * p.kv_splits;
    DCB_REQUIRE(blocks < (1ll << 31), "too many keys");
    const auto aligned = [&](const AttnTensor& t) {
        return reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.sc % 4 == 0 && (p.n == 1 || t.sn % 4 == 0);
    };
    const bool gather = p.kv_mask || p.sk % 4 != 0 || !aligned(p.k) || !aligned(p.v) || !aligned(p.dk) || !aligned(p.dv);
    const auto sized = [&](auto w) -> int32_t {
        constexpr int WARPS = decltype(w)::value;
        DCB_CUDA_TRY(launch_overlapped(gather ? attn_thin_bwd_kernel<WARPS, true> : attn_thin_bwd_kernel<WARPS, false>,
                                       dim3((unsigned) blocks), 32 * WARPS, 0, stream, p));
        return DCB_OK;
    };
    if (p.d <= 32)
        return sized(std::integral_constant<int, 4>());
    if (p.d <= 64)
        return sized(std::integral_constant<int, 8>());
    return sized(std::integral_constant<int, 16>());
}

int32_t attn_thin_fwd(const AttnProblem& p, int32_t dtype, cudaStream_t stream)
{
    return dtype == DCB_BF16 ? ath_fwd<bf16>(p, stream) : ath_fwd<float>(p, stream);
}

} // namespace dcb
