// Attention of fp32 tensors on the CUDA cores, forward and backward.
//
// Blocks of 256 threads hold tiles of 64 cells as [channel][cell], as memory has them.  A thread
// has 4 x 4 scores of a 64 x 64 tile (outer products over the channels) and 4 cells x D / 16
// channels of the result (products over the tile's other cells).  The forward pass keeps the
// running maximum and sum of a row beside its result; the backward pass works the weights out
// again from lse, once by tiles of keys (dk, dv) and once by tiles of queries (dq), so that every
// result has one owner and its sums one order.
//
// Bound by the fp32 pipes and shared memory: 2 x 8 heads of 64 on 32^2 cells take 155 us forward (28 TFLOP/s), 368 and
// 221 us backward.  From 65 channels on the backward kernels' tiles leave room for one block an SM, and wait more: 8 heads of
// 128, 2 key heads, 40 x 55 cells, a training step 3.1 ms (22 TFLOP/s).
#include "attention.cuh"

namespace dcb
{
namespace
{

constexpr int AS_TILE = 64;
constexpr int AS_PITCH = 68; // floats: rows 16-byte aligned, four rows on different banks
constexpr int AS_THREADS = 256;

// One head's cells, 64 from the r0-th on of those that are there, to shared memory as [channel][cell]; cells that are not,
// and channels up to D, as zeros.
template <int D>
__device__ __forceinline__ void as_load(float* to, const AttnTensor& t, long long n, int head, int d, int r0,
                                        const AttnCells& cells)
{
    const int j = threadIdx.x & 63, c0 = threadIdx.x >> 6;
    const bool in = r0 + j < cells.count;
    const float* p = static_cast<const float*>(t.p) + n * t.sn + ((long long) head * d + c0) * t.sc
                     + (in ? cells.cell(r0 + j) : 0);
    // eight loads go out before the first is waited for
#pragma unroll
    for (int k0 = 0; k0 < D / 4; k0 += 8)
    {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v[k] = in && c0 + 4 * (k0 + k) < d ? p[4 * (k0 + k) * t.sc] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            to[(c0 + 4 * (k0 + k)) * AS_PITCH + j] = v[k];
    }
}

// s[a][b] = sum_c A[c][4 ty + a] B[c][4 tx + b]
template <int D>
__device__ __forceinline__ void as_scores(const float* A, const float* B, int tx, int ty, float (&s)[4][4])
{
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            s[a][b] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; ++c)
    {
        float x[4], y[4];
        load_elems<4>(A + c * AS_PITCH + 4 * ty, x);
        load_elems<4>(B + c * AS_PITCH + 4 * tx, y);
#pragma unroll
        for (int a = 0; a < 4; ++a)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                s[a][b] = fmaf(x[a], y[b], s[a][b]);
    }
}

// Row t of a tile of weights lies at as_row(t): the rows that neighbouring threads write are neighbours then, four banks
// apart, and are written as 16 bytes.
__device__ __forceinline__ int as_row(int t)
{
    return ((t & 3) * 16 + (t >> 2)) * AS_PITCH;
}

// acc[e][r] += sum_t W[t][4 ty + e] X[tx + 16 r][t].  A tile's 64 terms are added up by themselves first: over n tiles a
// result is then off by at most (64 + n) roundings, not 64 n.  (2^25 keys of equal weight: 1.7e-3 of the result otherwise.)
template <int D>
__device__ __forceinline__ void as_accumulate(const float* W, const float* X, int tx, int ty, float (&acc)[4][D / 16])
{
    float sum[4][D / 16];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            sum[e][r] = 0.f;
#pragma unroll 2
    for (int t = 0; t < AS_TILE; t += 4)
    {
        float w[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            load_elems<4>(W + as_row(t + u) + 4 * ty, w[u]);
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
        {
            float x[4];
            load_elems<4>(X + (tx + 16 * r) * AS_PITCH + t, x);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sum[e][r] = fmaf(w[u][e], x[u], sum[e][r]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            acc[e][r] += sum[e][r];
}

// Results of 4 cells x D / 16 channels: to the tensor, or as a part to [head][channel][cell].
template <int D>
__device__ __forceinline__ void as_store(const AttnTensor& t, float* part, long long nh, long long n, int head, int d,
                                         int r0, const AttnCells& side, int tx, int ty, const float (&acc)[4][D / 16])
{
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        const int row = r0 + 4 * ty + e;
        if (row >= side.count)
            continue;
        const int i = side.cell(row);
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
        {
            const int c = tx + 16 * r;
            if (c < d)
                (part ? part + (nh * d + c) * side.cells
                      : static_cast<float*>(t.p) + n * t.sn + ((long long) head * d + c) * t.sc)[i]
                    = acc[e][r];
        }
    }
}

// A thread's 4 x 4 scores as rows 4 tx ... of a tile [key][query].
__device__ __forceinline__ void as_put_by_column(float* W, int tx, int ty, const float (&s)[4][4])
{
#pragma unroll
    for (int b = 0; b < 4; ++b)
    {
        const float v[4] = {s[0][b], s[1][b], s[2][b], s[3][b]};
        store_elems<4>(W + as_row(4 * tx + b) + 4 * ty, v);
    }
}

struct AsAt
{
    int tile, split;
    long long nh, n;
    int head;
};

__device__ __forceinline__ AsAt as_at(int tiles, int splits, int heads)
{
    AsAt a;
    long long b = blockIdx.x;
    a.tile = tiles - 1 - (int) (b % tiles); // causal: the longest walks first
    b /= tiles;
    a.split = (int) (b % splits);
    a.nh = b / splits;
    a.n = a.nh / heads;
    a.head = (int) (a.nh - a.n * heads);
    return a;
}

// Part `split` of `steps` tiles.
__device__ __forceinline__ void as_range(int steps, int splits, int split, int* lo, int* hi)
{
    *lo = (int) ((long long) steps * split / splits);
    *hi = (int) ((long long) steps * (split + 1) / splits);
}

template <int D>
__global__ void __launch_bounds__(AS_THREADS) attn_simt_fwd_kernel(AttnProblem p)
{
    extern __shared__ float smem[];
    float *Q = smem, *K = Q + D * AS_PITCH, *V = K + D * AS_PITCH, *P = V + D * AS_PITCH;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const AsAt at = as_at(attn_tiles(p.sq, AS_TILE), p.kv_splits, p.q_heads);
    const int i0 = at.tile * AS_TILE, kv_head = at.head / p.group;
    const AttnCells q(p.q_side, at.n, p.sq), kv(p.kv_side, at.n, p.sk);
    if (i0 >= q.count)
        return;
    as_load<D>(Q, p.q, at.n, at.head, p.d, i0, q);
    int limit[4]; // keys that a row sees
#pragma unroll
    for (int a = 0; a < 4; ++a)
        limit[a] = attn_limit(p, q, kv, i0 + 4 * ty + a);
    float m[4], l[4], acc[4][D / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a)
    {
        m[a] = -INFINITY, l[a] = 0.f;
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            acc[a][r] = 0.f;
    }
    int lo, hi;
    as_range(attn_tiles(kv.count, AS_TILE), p.kv_splits, at.split, &lo, &hi);
    hi = min(hi, attn_tiles(attn_limit(p, q, kv, min(i0 + AS_TILE, q.count) - 1), AS_TILE));
    for (int t = lo; t < hi; ++t)
    {
        const int j0 = t * AS_TILE;
        __syncthreads();
        as_load<D>(K, p.k, at.n, kv_head, p.d, j0, kv);
        as_load<D>(V, p.v, at.n, kv_head, p.d, j0, kv);
        __syncthreads();
        float s[4][4];
        as_scores<D>(Q, K, tx, ty, s);
#pragma unroll
        for (int a = 0; a < 4; ++a)
        {
            float top = m[a];
#pragma unroll
            for (int b = 0; b < 4; ++b)
            {
                s[a][b] = j0 + 4 * tx + b < limit[a] ? s[a][b] * p.scale : -INFINITY;
                top = fmaxf(top, s[a][b]);
            }
#pragma unroll
            for (int h = 8; h >= 1; h /= 2)
                top = fmaxf(top, __shfl_xor_sync(~0u, top, h));
            const float base = top == -INFINITY ? 0.f : top, shrink = exp2f(m[a] - base);
            m[a] = top;
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < 4; ++b)
            {
                s[a][b] = exp2f(s[a][b] - base);
                sum += s[a][b];
            }
#pragma unroll
            for (int h = 8; h >= 1; h /= 2)
                sum += __shfl_xor_sync(~0u, sum, h);
            l[a] = fmaf(l[a], shrink, sum);
#pragma unroll
            for (int r = 0; r < D / 16; ++r)
                acc[a][r] *= shrink;
        }
        as_put_by_column(P, tx, ty, s);
        __syncthreads();
        as_accumulate<D>(P, V, tx, ty, acc);
    }
    const long long heads = (long long) p.n * p.q_heads;
    if (p.kv_splits > 1)
    {
        if (tx == 0)
#pragma unroll
            for (int a = 0; a < 4; ++a)
                if (i0 + 4 * ty + a < q.count)
                {
                    float* ml = p.part_ml + (2 * heads * at.split + at.nh) * p.sq + q.cell(i0 + 4 * ty + a);
                    ml[0] = m[a];
                    ml[heads * p.sq] = l[a];
                }
        as_store<D>(p.o, p.part_o + at.split * heads * p.d * p.sq, at.nh, at.n, at.head, p.d, i0, q, tx, ty,
                    acc);
        return;
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
    {
        const int i = i0 + 4 * ty + a;
        const bool none = l[a] == 0.f;
        const float f = none ? 0.f : 1.f / l[a];
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            acc[a][r] = none ? 0.f : acc[a][r] * f;
        if (tx == 0 && i < q.count)
            p.lse[at.nh * p.sq + q.cell(i)] = none ? -INFINITY : (m[a] + log2f(l[a])) / ATTN_LOG2E;
    }
    as_store<D>(p.o, nullptr, at.nh, at.n, at.head, p.d, i0, q, tx, ty, acc);
}

// The weights and their gradients of a tile, P = exp2(s - lse), dS = P (dP - delta): [query][key] or [key][query].
template <int D, bool BY_KEY>
__device__ __forceinline__ void as_weights(const AttnProblem& p, const float* Q, const float* K, const float* V,
                                           const float* dO, const float* lse, const float* delta,
                                           const int* limit, int j0, int tx, int ty, float* P, float* dS)
{
    float s[4][4], dp[4][4];
    as_scores<D>(Q, K, tx, ty, s);
    as_scores<D>(dO, V, tx, ty, dp);
#pragma unroll
    for (int a = 0; a < 4; ++a)
    {
        const int i = 4 * ty + a;
        const float top = lse[i], del = delta[i];
        const int seen = limit[i];
#pragma unroll
        for (int b = 0; b < 4; ++b)
        {
            const float w = j0 + 4 * tx + b < seen ? exp2f(fmaf(s[a][b], p.scale, -top)) : 0.f;
            dp[a][b] = w == 0.f ? 0.f : w * (dp[a][b] - del);
            s[a][b] = w;
        }
        if (BY_KEY) // [query][key]
        {
            store_elems<4>(P + as_row(i) + 4 * tx, s[a]);
            store_elems<4>(dS + as_row(i) + 4 * tx, dp[a]);
        }
    }
    if (!BY_KEY)
        as_put_by_column(dS, tx, ty, dp);
}

__device__ __forceinline__ void as_load_stats(const AttnProblem& p, const AttnCells& q, const AttnCells& kv,
                                              long long nh, int i0, float* lse, float* delta, int* limit)
{
    if (threadIdx.x < AS_TILE)
    {
        const int i = i0 + threadIdx.x;
        limit[threadIdx.x] = attn_limit(p, q, kv, i);
        lse[threadIdx.x] = i < q.count ? p.stats[nh * p.stats_pitch + i] : INFINITY;
        delta[threadIdx.x] = i < q.count ? p.stats[((long long) p.n * p.q_heads + nh) * p.stats_pitch + i] : 0.f;
    }
}

template <int D>
__global__ void __launch_bounds__(AS_THREADS) attn_simt_dkv_kernel(AttnProblem p)
{
    extern __shared__ float smem[];
    float *K = smem, *V = K + D * AS_PITCH, *Q = V + D * AS_PITCH, *dO = Q + D * AS_PITCH, *P = dO + D * AS_PITCH,
          *dS = P + AS_TILE * AS_PITCH;
    __shared__ float lse[AS_TILE], delta[AS_TILE];
    __shared__ int limit[AS_TILE];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const AsAt at = as_at(attn_tiles(p.sk, AS_TILE), p.q_splits, p.kv_heads);
    const int j0 = at.tile * AS_TILE;
    const AttnCells q(p.q_side, at.n, p.sq), kv(p.kv_side, at.n, p.sk);
    if (j0 >= kv.count)
        return;
    as_load<D>(K, p.k, at.n, at.head, p.d, j0, kv);
    as_load<D>(V, p.v, at.n, at.head, p.d, j0, kv);
    float gk[4][D / 16], gv[4][D / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            gk[a][r] = gv[a][r] = 0.f;
    // tiles of queries from the first that sees a key of this tile on, of every query head of the group
    const int t0 = p.causal ? q.before((long long) kv.cell(j0) - p.offset) / AS_TILE : 0;
    const int tiles = max(0, attn_tiles(q.count, AS_TILE) - t0);
    int lo, hi;
    as_range(tiles * p.group, p.q_splits, at.split, &lo, &hi);
    for (int u = lo; u < hi; ++u)
    {
        const int g = u / tiles, i0 = (t0 + u - g * tiles) * AS_TILE, head = at.head * p.group + g;
        __syncthreads();
        as_load<D>(Q, p.q, at.n, head, p.d, i0, q);
        as_load<D>(dO, p.d_o, at.n, head, p.d, i0, q);
        as_load_stats(p, q, kv, at.n * p.q_heads + head, i0, lse, delta, limit);
        __syncthreads();
        as_weights<D, true>(p, Q, K, V, dO, lse, delta, limit, j0, tx, ty, P, dS);
        __syncthreads();
        as_accumulate<D>(P, dO, tx, ty, gv);
        as_accumulate<D>(dS, Q, tx, ty, gk);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            gk[a][r] *= p.scale / ATTN_LOG2E;
    const long long size = (long long) p.n * p.kv_heads * p.d * p.sk * at.split;
    as_store<D>(p.dk, p.q_splits > 1 ? p.part_dk + size : nullptr, at.nh, at.n, at.head, p.d, j0, kv, tx, ty, gk);
    as_store<D>(p.dv, p.q_splits > 1 ? p.part_dv + size : nullptr, at.nh, at.n, at.head, p.d, j0, kv, tx, ty, gv);
}

template <int D>
__global__ void __launch_bounds__(AS_THREADS) attn_simt_dq_kernel(AttnProblem p)
{
    extern __shared__ float smem[];
    float *Q = smem, *dO = Q + D * AS_PITCH, *K = dO + D * AS_PITCH, *V = K + D * AS_PITCH, *dS = V + D * AS_PITCH;
    __shared__ float lse[AS_TILE], delta[AS_TILE];
    __shared__ int limit[AS_TILE];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const AsAt at = as_at(attn_tiles(p.sq, AS_TILE), p.kv_splits, p.q_heads);
    const int i0 = at.tile * AS_TILE, kv_head = at.head / p.group;
    const AttnCells q(p.q_side, at.n, p.sq), kv(p.kv_side, at.n, p.sk);
    if (i0 >= q.count)
        return;
    as_load<D>(Q, p.q, at.n, at.head, p.d, i0, q);
    as_load<D>(dO, p.d_o, at.n, at.head, p.d, i0, q);
    as_load_stats(p, q, kv, at.nh, i0, lse, delta, limit);
    float gq[4][D / 16];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            gq[a][r] = 0.f;
    int lo, hi;
    as_range(attn_tiles(kv.count, AS_TILE), p.kv_splits, at.split, &lo, &hi);
    hi = min(hi, attn_tiles(attn_limit(p, q, kv, min(i0 + AS_TILE, q.count) - 1), AS_TILE));
    for (int t = lo; t < hi; ++t)
    {
        const int j0 = t * AS_TILE;
        __syncthreads();
        as_load<D>(K, p.k, at.n, kv_head, p.d, j0, kv);
        as_load<D>(V, p.v, at.n, kv_head, p.d, j0, kv);
        __syncthreads();
        as_weights<D, false>(p, Q, K, V, dO, lse, delta, limit, j0, tx, ty, nullptr, dS);
        __syncthreads();
        as_accumulate<D>(dS, K, tx, ty, gq);
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < D / 16; ++r)
            gq[a][r] *= p.scale / ATTN_LOG2E;
    float* part = p.kv_splits > 1 ? p.part_dq + (long long) at.split * p.n * p.q_heads * p.d * p.sq : nullptr;
    as_store<D>(p.dq, part, at.nh, at.n, at.head, p.d, i0, q, tx, ty, gq);
}

int32_t as_launch(void (*kernel)(AttnProblem), const AttnProblem& p, long long blocks, int smem, cudaStream_t stream)
{
    DCB_REQUIRE(blocks < (1ll << 31), "too many tiles");
    if (blocks == 0)
        return DCB_OK;
    if (int32_t e = allow_dynamic_smem((const void*) kernel, smem))
        return e;
    kernel<<<(unsigned) blocks, AS_THREADS, smem, stream>>>(p);
    DCB_LAUNCH_CHECK();
    return DCB_OK;
}

template <class F>
int32_t as_with(int d, F f)
{
    if (d <= 32)
        return f(std::integral_constant<int, 32>());
    if (d <= 64)
        return f(std::integral_constant<int, 64>());
    return f(std::integral_constant<int, 128>());
}

} // namespace

// Parts of a walk over `steps` tiles, for `work` walks of which `slots` go at a time: how many rounds there are, and how
// long one takes, start and end of a block counted as a tile.
static int as_parts(long long work, int steps, long long slots)
{
    int best = 1;
    long long least = 0;
    for (int s = 1; s <= std::min(steps, 64); ++s)
    {
        const long long cost = (work * s + slots - 1) / slots * (attn_tiles(steps, s) + 1);
        if (s == 1 || 100 * cost < 97 * least)
            best = s, least = cost;
    }
    return best;
}

void attn_simt_splits(AttnProblem* p, bool backward)
{
    const long long slots = (p->d <= 64 ? 2ll : 1ll) * num_sms(); // blocks an SM has room for
    const int left = p->q_mask || p->kv_mask ? 2 : 1; // masks are taken to leave half of either side
    const int q_tiles = attn_tiles(p->sq, AS_TILE), k_tiles = attn_tiles(p->sk, AS_TILE);
    // Causal walks differ in length: parts enough for three blocks an SM (two of 64 channels) even them out.  4 heads of
    // 96, 40 x 55 cells, causal, forward 266 us, by rounds 379; 4 heads of 128, 2 key heads, 40 x 41, 242 by rounds, 292
    // with parts for two blocks an SM.
    const auto parts = [&](long long work, int steps) {
        work = (work + left - 1) / left, steps /= left;
        return p->causal ? attn_splits(work, steps, (p->d <= 64 ? 2ll : 3ll) * num_sms()) : as_parts(work, steps, slots);
    };
    p->kv_splits = parts((long long) p->n * p->q_heads * q_tiles, k_tiles);
    p->q_splits = backward ? parts((long long) p->n * p->kv_heads * k_tiles, q_tiles * p->group) : 1;
}

int32_t attn_simt_fwd(const AttnProblem& p, cudaStream_t stream)
{
    return as_with(p.d, [&](auto d) {
        constexpr int D = decltype(d)::value;
        return as_launch(attn_simt_fwd_kernel<D>, p,
                         (long long) p.n * p.q_heads * attn_tiles(p.sq, AS_TILE) * p.kv_splits,
                         (3 * D + AS_TILE) * AS_PITCH * 4, stream);
    });
}

int32_t attn_simt_bwd(const AttnProblem& p, cudaStream_t stream)
{
    return as_with(p.d, [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (int32_t e = as_launch(attn_simt_dkv_kernel<D>, p,
                                  (long long) p.n * p.kv_heads * attn_tiles(p.sk, AS_TILE) * p.q_splits,
                                  (4 * D + 2 * AS_TILE) * AS_PITCH * 4, stream))
            return e;
        return as_launch(attn_simt_dq_kernel<D>, p,
                         (long long) p.n * p.q_heads * attn_tiles(p.sq, AS_TILE) * p.kv_splits,
                         (4 * D + AS_TILE) * AS_PITCH * 4, stream);
    });
}

} // namespace dcb
