// Layer normalisation over the channels of every cell, forward and backward.
//
// In NC[D]HW a cell's channels lie a volume apart, its neighbours in W beside it.  A warp's
// lanes therefore take neighbouring units of V cells, and a cell's C channels are dealt out to
// the G warps of a group, K each: all accesses are coalesced, a tensor is read once and kept in
// registers, and what the warps of a group exchange is two floats a cell (their sum and their
// centred sum of squares forward, the two sums of the gradient backward).  HBM bound: 2 tensors
// forward, 3 backward.
#include "elem.cuh"

namespace dcb
{
namespace
{

constexpr int LN_WIDE_WARPS = 16;  // warps of a block of the kernels for many channels
constexpr int LN_CHUNK = 32;       // channels that a lane of those takes at a time
constexpr int LN_MAX_GROUP = 16;   // warps of a group: 512 threads of up to 128 registers
constexpr int LN_NARROW = LN_MAX_GROUP * 32;
constexpr int LN_MAX_CHANNELS = 16384; // the wide backward kernel's sums fill 128 KB of shared memory

struct LnGeom
{
    CellUnits units;
    long long per_run, rows, rows_inner;
    int c, g;         // channels; warps of a group
    long long tiles;  // of 32 units a group of warps
};

__device__ __forceinline__ CellAt ln_cell(const LnGeom& g, long long unit, int v)
{
    return v == 4   ? cell_at<4>(g.units, g.per_run, g.rows, g.rows_inner, unit)
           : v == 2 ? cell_at<2>(g.units, g.per_run, g.rows, g.rows_inner, unit)
                    : cell_at<1>(g.units, g.per_run, g.rows, g.rows_inner, unit);
}

// Sum and centred sum of squares of all channels from those of the groups' parts (Chan et al.): no cancellation
// between large squares, whatever the mean.
template <int V>
__device__ __forceinline__ void ln_join(const float* part, int g, int c, int lane, float (&mean)[V], float (&m2)[V])
{
    float s[V], q[V], t[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
        s[e] = 0.f;
    for (int i = 0; i < g; ++i)
    {
        load_elems<V>(part + (2 * i * 32 + lane) * V, t);
#pragma unroll
        for (int e = 0; e < V; ++e)
            s[e] += t[e];
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        mean[e] = s[e] / c, m2[e] = 0.f;
    for (int i = 0; i < g; ++i)
    {
        const int count = (c - i + g - 1) / g;
        load_elems<V>(part + (2 * i * 32 + lane) * V, t);
        load_elems<V>(part + ((2 * i + 1) * 32 + lane) * V, q);
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            const float d = t[e] / count - mean[e];
            m2[e] += q[e] + count * d * d;
        }
    }
}

template <class T, int V, int K>
__global__ void __launch_bounds__(512)
    ln_fwd_kernel(const T* x, RunStrides xs, T* y, RunStrides ys, const float* scale, const float* bias, float eps,
                  float* mean_out, float* inv_std_out, LnGeom geo)
{
    extern __shared__ float part[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = warp / geo.g, cg = warp - group * geo.g;
    wait_for_previous_kernel(x, scale, bias);
    dependents_may_start();
    const long long unit = ((long long) blockIdx.x * (blockDim.x / 32 / geo.g) + group) * 32 + lane;
    const bool live = unit < geo.units.total;
    CellAt at = {};
    float v[K][V];
    if (live)
    {
        at = ln_cell(geo, unit, V);
        const T* px = x + offset_of(at, xs);
#pragma unroll
        for (int k = 0; k < K; ++k)
        {
            const int c = cg + k * geo.g;
            if (c < geo.c)
                load_elems<V>(px + c * xs.sc, v[k]);
        }
    }
    const int count = (geo.c - cg + geo.g - 1) / geo.g; // at least 1: g <= c
    float sum[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
    {
        sum[e] = m2[e] = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < count)
                sum[e] += live ? v[k][e] : 0.f;
        const float m = sum[e] / count;
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (k < count)
            {
                const float d = (live ? v[k][e] : 0.f) - m;
                m2[e] = fmaf(d, d, m2[e]);
            }
    }
    float mean[V];
    if (geo.g > 1)
    {
        float* mine = part + group * geo.g * 2 * 32 * V;
        store_elems<V>(mine + (2 * cg * 32 + lane) * V, sum);
        store_elems<V>(mine + ((2 * cg + 1) * 32 + lane) * V, m2);
        __syncthreads();
        ln_join<V>(mine, geo.g, geo.c, lane, mean, m2);
    }
    else
    {
#pragma unroll
        for (int e = 0; e < V; ++e)
            mean[e] = sum[e] / count;
    }
    if (!live)
        return;
    float inv[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
        inv[e] = 1.f / sqrtf(m2[e] / geo.c + eps);
    if (cg == 0)
    {
        const long long i = at.n * geo.units.cells + at.cell;
        if (mean_out)
            store_elems<V>(mean_out + i, mean);
        if (inv_std_out)
            store_elems<V>(inv_std_out + i, inv);
    }
    T* py = y + offset_of(at, ys);
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        const int c = cg + k * geo.g;
        if (c < geo.c)
        {
            const float w = scale ? scale[c] : 1.f, b = bias ? bias[c] : 0.f;
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
                out[e] = fmaf((v[k][e] - mean[e]) * inv[e], w, b);
            store_elems<V>(py + c * ys.sc, out);
        }
    }
}

// Sums over a warp's lanes of K values a lane, by halves: lane l ends with the sum of value l mod K
// in v[0].  K - 1 + log2(32 / K) exchanges instead of 5 K.
template <int K>
__device__ __forceinline__ float ln_lane_sums(float (&v)[K], int lane)
{
#pragma unroll
    for (int h = K / 2; h >= 1; h /= 2)
    {
        const bool upper = lane & h;
#pragma unroll
        for (int i = 0; i < h; ++i)
        {
            const float send = upper ? v[i] : v[i + h];
            const float keep = upper ? v[i + h] : v[i];
            v[i] = keep + __shfl_xor_sync(~0u, send, h);
        }
    }
    float r = v[0];
#pragma unroll
    for (int h = K; h < 32; h *= 2)
        r += __shfl_xor_sync(~0u, r, h);
    return r;
}

// Blocks walk over the tiles; the gradients of scale and bias stay in registers, K channels a
// lane, and are added up over the lanes once, at the end: partial[which][channel][block].
template <class T, int V, int K>
__global__ void __launch_bounds__(512)
    ln_bwd_kernel(const T* x, RunStrides xs, const T* dy, RunStrides dys, const float* mean_in,
                  const float* inv_std_in, const float* scale, T* dx, RunStrides dxs, float* partial, LnGeom geo)
{
    extern __shared__ float part[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int groups = blockDim.x / 32 / geo.g;
    const int group = warp / geo.g, cg = warp - group * geo.g;
    const int stage = groups * geo.g * 2 * 32 * V;
    wait_for_previous_kernel(x, dy, mean_in, inv_std_in, scale);
    dependents_may_start();
    float acc_w[K], acc_b[K], w[K];
#pragma unroll
    for (int k = 0; k < K; ++k)
    {
        acc_w[k] = acc_b[k] = 0.f;
        const int c = cg + k * geo.g;
        w[k] = scale && c < geo.c ? scale[c] : 1.f;
    }
    int turn = 0;
    for (long long tile = blockIdx.x; tile < geo.tiles; tile += gridDim.x, turn ^= 1)
    {
        const long long unit = (tile * groups + group) * 32 + lane;
        const bool live = unit < geo.units.total;
        CellAt at = {};
        float u[K][V], d[K][V], mean[V], inv[V], a[V], b[V];
        if (live)
        {
            at = ln_cell(geo, unit, V);
            const T* px = x + offset_of(at, xs);
            const T* pd = dy + offset_of(at, dys);
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                const int c = cg + k * geo.g;
                if (c < geo.c)
                {
                    load_elems<V>(px + c * xs.sc, u[k]);
                    load_elems<V>(pd + c * dys.sc, d[k]);
                }
            }
            load_elems<V>(mean_in + at.n * geo.units.cells + at.cell, mean);
            load_elems<V>(inv_std_in + at.n * geo.units.cells + at.cell, inv);
        }
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            a[e] = b[e] = 0.f;
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                const bool have = live && cg + k * geo.g < geo.c;
                u[k][e] = have ? (u[k][e] - mean[e]) * inv[e] : 0.f;
                d[k][e] = have ? d[k][e] : 0.f;
                acc_w[k] = fmaf(d[k][e], u[k][e], acc_w[k]);
                acc_b[k] += d[k][e];
                const float g = d[k][e] * w[k];
                a[e] += g;
                b[e] = fmaf(g, u[k][e], b[e]);
            }
        }
        if (geo.g > 1)
        {
            float* mine = part + turn * stage + group * geo.g * 2 * 32 * V;
            store_elems<V>(mine + (2 * cg * 32 + lane) * V, a);
            store_elems<V>(mine + ((2 * cg + 1) * 32 + lane) * V, b);
            __syncthreads(); // the other half of `part` is free again behind the next tile's barrier
#pragma unroll
            for (int e = 0; e < V; ++e)
                a[e] = b[e] = 0.f;
            for (int i = 0; i < geo.g; ++i)
            {
                float s[V], t[V];
                load_elems<V>(mine + (2 * i * 32 + lane) * V, s);
                load_elems<V>(mine + ((2 * i + 1) * 32 + lane) * V, t);
#pragma unroll
                for (int e = 0; e < V; ++e)
                    a[e] += s[e], b[e] += t[e];
            }
        }
        if (live)
        {
#pragma unroll
            for (int e = 0; e < V; ++e)
                a[e] /= geo.c, b[e] /= geo.c;
            T* po = dx + offset_of(at, dxs);
#pragma unroll
            for (int k = 0; k < K; ++k)
            {
                const int c = cg + k * geo.g;
                if (c < geo.c)
                {
                    float out[V];
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        out[e] = inv[e] * (fmaf(d[k][e], w[k], -a[e]) - u[k][e] * b[e]);
                    store_elems<V>(po + c * dxs.sc, out);
                }
            }
        }
    }
    if (!partial)
        return;
    // groups of a block first, in order, then the lanes
    const float sw = ln_lane_sums<K>(acc_w, lane), sb = ln_lane_sums<K>(acc_b, lane);
    __syncthreads();
    const int slots = geo.g * K;
    if (lane < K)
    {
        part[(group * 2) * slots + cg + lane * geo.g] = sw;
        part[(group * 2 + 1) * slots + cg + lane * geo.g] = sb;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * geo.c; i += blockDim.x)
    {
        const int which = i >= geo.c, c = which ? i - geo.c : i;
        float s = 0.f;
        for (int p = 0; p < groups; ++p)
            s += part[(p * 2 + which) * slots + c];
        partial[(long long) i * gridDim.x + blockIdx.x] = s;
    }
}

// More channels than a block's registers hold: the cell's channels are read twice, the second time from L2 (a
// block's tile of 32 cells is 128 bytes a channel).
template <class T>
__global__ void __launch_bounds__(32 * LN_WIDE_WARPS)
    ln_fwd_wide_kernel(const T* x, RunStrides xs, T* y, RunStrides ys, const float* scale, const float* bias,
                       float eps, float* mean_out, float* inv_std_out, LnGeom geo)
{
    __shared__ float part[2][LN_WIDE_WARPS][2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (geo.c + LN_CHUNK - 1) / LN_CHUNK;
    wait_for_previous_kernel(x, scale, bias);
    dependents_may_start();
    int turn = 0;
    for (long long tile = blockIdx.x; tile < geo.tiles; tile += gridDim.x, turn ^= 1)
    {
        const long long unit = tile * 32 + lane;
        const bool live = unit < geo.units.total;
        const CellAt at = ln_cell(geo, live ? unit : 0, 1);
        const T* px = x + offset_of(at, xs);
        float mean = 0.f, m2 = 0.f;
        int have = 0;
        for (int q = warp; q < chunks; q += LN_WIDE_WARPS)
        {
            const int c0 = q * LN_CHUNK, count = min(LN_CHUNK, geo.c - c0);
            float v[LN_CHUNK][1], s = 0.f, t = 0.f;
#pragma unroll
            for (int k = 0; k < LN_CHUNK; ++k)
                if (k < count)
                    load_elems<1>(px + (c0 + k) * xs.sc, v[k]);
#pragma unroll
            for (int k = 0; k < LN_CHUNK; ++k)
                if (k < count)
                    s += v[k][0];
            s /= count;
#pragma unroll
            for (int k = 0; k < LN_CHUNK; ++k)
                if (k < count)
                    t = fmaf(v[k][0] - s, v[k][0] - s, t);
            const float d = s - mean;
            m2 += t + d * d * ((float) have * count / (have + count));
            mean += d * count / (have + count);
            have += count;
        }
        part[turn][warp][0][lane] = mean;
        part[turn][warp][1][lane] = m2;
        __syncthreads();
        mean = m2 = 0.f;
        have = 0;
        for (int i = 0; i < LN_WIDE_WARPS; ++i)
        {
            int count = 0; // channels of warp i
            for (int q = i; q < chunks; q += LN_WIDE_WARPS)
                count += min(LN_CHUNK, geo.c - q * LN_CHUNK);
            if (count == 0)
                break;
            const float d = part[turn][i][0][lane] - mean;
            m2 += part[turn][i][1][lane] + d * d * ((float) have * count / (have + count));
            mean += d * count / (have + count);
            have += count;
        }
        if (!live)
            continue;
        const float inv = 1.f / sqrtf(m2 / geo.c + eps);
        if (warp == 0)
        {
            const long long i = at.n * geo.units.cells + at.cell;
            if (mean_out)
                mean_out[i] = mean;
            if (inv_std_out)
                inv_std_out[i] = inv;
        }
        T* py = y + offset_of(at, ys);
        for (int q = warp; q < chunks; q += LN_WIDE_WARPS)
        {
            const int c0 = q * LN_CHUNK, count = min(LN_CHUNK, geo.c - c0);
            float v[LN_CHUNK][1];
#pragma unroll
            for (int k = 0; k < LN_CHUNK; ++k)
                if (k < count)
                    load_elems<1>(px + (c0 + k) * xs.sc, v[k]);
#pragma unroll
            for (int k = 0; k < LN_CHUNK; ++k)
                if (k < count)
                {
                    const int c = c0 + k;
                    float out[1] = {fmaf((v[k][0] - mean) * inv, scale ? scale[c] : 1.f, bias ? bias[c] : 0.f)};
                    store_elems<1>(py + c * ys.sc, out);
                }
        }
    }
}

template <class T>
__global__ void __launch_bounds__(32 * LN_WIDE_WARPS)
    ln_bwd_wide_kernel(const T* x, RunStrides xs, const T* dy, RunStrides dys, const float* mean_in,
                       const float* inv_std_in, const float* scale, T* dx, RunStrides dxs, float* partial, LnGeom geo)
{
    extern __shared__ float acc[]; // [2][c]: a channel belongs to one warp
    __shared__ float part[2][LN_WIDE_WARPS][2][32];
    constexpr int HALF = LN_CHUNK / 2; // channels at a time: x and dy are both held
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = (geo.c + HALF - 1) / HALF;
    for (int i = threadIdx.x; i < 2 * geo.c; i += blockDim.x)
        acc[i] = 0.f;
    wait_for_previous_kernel(x, dy, mean_in, inv_std_in, scale);
    dependents_may_start();
    __syncthreads();
    int turn = 0;
    for (long long tile = blockIdx.x; tile < geo.tiles; tile += gridDim.x, turn ^= 1)
    {
        const long long unit = tile * 32 + lane;
        const bool live = unit < geo.units.total;
        const CellAt at = ln_cell(geo, live ? unit : 0, 1);
        const T* px = x + offset_of(at, xs);
        const T* pd = dy + offset_of(at, dys);
        const float mean = mean_in[at.n * geo.units.cells + at.cell];
        const float inv = inv_std_in[at.n * geo.units.cells + at.cell];
        float a = 0.f, b = 0.f;
        for (int q = warp; q < chunks; q += LN_WIDE_WARPS)
        {
            const int c0 = q * HALF, count = min(HALF, geo.c - c0);
            float u[HALF][1], d[HALF][1], wu[HALF], wb[HALF];
#pragma unroll
            for (int k = 0; k < HALF; ++k)
                if (k < count)
                {
                    load_elems<1>(px + (c0 + k) * xs.sc, u[k]);
                    load_elems<1>(pd + (c0 + k) * dys.sc, d[k]);
                }
#pragma unroll
            for (int k = 0; k < HALF; ++k)
            {
                const bool use = live && k < count;
                const float uu = use ? (u[k][0] - mean) * inv : 0.f;
                const float dd = use ? d[k][0] : 0.f;
                const float g = dd * (scale && k < count ? scale[c0 + k] : 1.f);
                a += g;
                b = fmaf(g, uu, b);
                wu[k] = dd * uu;
                wb[k] = dd;
            }
            if (partial)
            {
                const float sw = ln_lane_sums<HALF>(wu, lane), sb = ln_lane_sums<HALF>(wb, lane);
                if (lane < count)
                {
                    acc[c0 + lane] += sw;
                    acc[geo.c + c0 + lane] += sb;
                }
            }
        }
        part[turn][warp][0][lane] = a;
        part[turn][warp][1][lane] = b;
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < LN_WIDE_WARPS; ++i)
            a += part[turn][i][0][lane], b += part[turn][i][1][lane];
        if (!live)
            continue;
        a /= geo.c;
        b /= geo.c;
        T* po = dx + offset_of(at, dxs);
        for (int q = warp; q < chunks; q += LN_WIDE_WARPS)
        {
            const int c0 = q * HALF, count = min(HALF, geo.c - c0);
            float u[HALF][1], d[HALF][1];
#pragma unroll
            for (int k = 0; k < HALF; ++k)
                if (k < count)
                {
                    load_elems<1>(px + (c0 + k) * xs.sc, u[k]);
                    load_elems<1>(pd + (c0 + k) * dys.sc, d[k]);
                }
#pragma unroll
            for (int k = 0; k < HALF; ++k)
                if (k < count)
                {
                    const float uu = (u[k][0] - mean) * inv;
                    float out[1] = {inv * (fmaf(d[k][0], scale ? scale[c0 + k] : 1.f, -a) - uu * b)};
                    store_elems<1>(po + (c0 + k) * dxs.sc, out);
                }
        }
    }
    if (!partial)
        return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * geo.c; i += blockDim.x)
        partial[(long long) i * gridDim.x + blockIdx.x] = acc[i];
}

// A warp a channel and gradient: the blocks' sums in order, in fp64.
__global__ void __launch_bounds__(256) ln_fold_kernel(const float* partial, int blocks, int c, float* dscale,
                                                      float* dbias)
{
    wait_for_previous_kernel(partial);
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const long long i = (long long) blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= 2ll * c)
        return;
    double s = 0.;
    for (int b = lane; b < blocks; b += 32)
        s += partial[i * blocks + b];
#pragma unroll
    for (int h = 16; h >= 1; h /= 2)
        s += __shfl_xor_sync(~0u, s, h);
    if (lane == 0)
        (i < c ? dscale + i : dbias + (i - c))[0] = (float) s;
}

__global__ void __launch_bounds__(256) ln_zero_kernel(float* dscale, float* dbias, int c)
{
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < c)
        dscale[i] = dbias[i] = 0.f;
}

// What a launch is made of: cells of an access, channels of a thread, warps of a group, groups of a block.
struct LnChoice
{
    int v, k, g, groups;
    bool wide;
};

LnChoice ln_choose(int c, int vmax, long long cells_of_all)
{
    LnChoice h = {1, 32, 1, 1, c > LN_NARROW};
    if (h.wide)
        return h;
    // V K = 32 values a thread.  Wide accesses first; fewer cells a thread where the tiles would not give every
    // SM two blocks, or where so many channels need more warps than a group has.
    for (int v = vmax; v >= 1; v /= 2)
    {
        h.v = v;
        h.k = v == 4 ? 8 : v == 2 ? 16 : 32;
        while (h.k > 4 && h.k / 2 >= c)
            h.k /= 2;
        h.g = (c + h.k - 1) / h.k;
        if (v == 1 || (h.g <= LN_MAX_GROUP && cells_of_all >= 2ll * num_sms() * 32 * v))
            break;
    }
    while (h.k > 4 && (c + h.k / 2 - 1) / (h.k / 2) <= 8) // small K, more warps: up to 8 to a group
    {
        h.k /= 2;
        h.g = (c + h.k - 1) / h.k;
    }
    h.groups = h.g >= 8 ? 1 : 8 / h.g;
    return h;
}

long long ln_blocks_max()
{
    return 8ll * num_sms();
}

int32_t ln_check(const dcb_nd_desc* xd, int32_t dtype)
{
    if (int32_t e = check_nd_desc(xd))
        return e;
    DCB_REQUIRE(known_dtype(dtype), "dtype must be DCB_F32 or DCB_BF16");
    DCB_REQUIRE(xd->c >= 1, "a cell needs a channel");
    if (xd->c > LN_MAX_CHANNELS)
    {
        set_last_error("unsupported: more than 16384 channels");
        return DCB_UNSUPPORTED;
    }
    return DCB_OK;
}

bool ln_empty(const dcb_nd_desc* d)
{
    return d->n == 0 || d->dims[0] == 0 || d->dims[1] == 0 || d->dims[2] == 0;
}

// Runs that all tensors of a call have; -1 where W is not dense in one of them.
int ln_level(std::initializer_list<const dcb_nd_desc*> ds)
{
    int level = 2;
    for (const dcb_nd_desc* d : ds)
        level = std::min(level, run_level(*d));
    return level;
}

template <class F>
int32_t ln_with_types(int32_t dtype, F f)
{
    return dtype == DCB_BF16 ? f(bf16()) : f(float());
}

LnGeom ln_geometry(const RunGeom& rg, const LnChoice& h)
{
    LnGeom g;
    g.units = cell_units(rg, h.v);
    g.per_run = rg.len / h.v;
    g.rows = rg.rows;
    g.rows_inner = rg.rows_inner;
    g.c = (int) rg.c;
    g.g = h.g;
    g.tiles = (g.units.total + 32ll * h.groups - 1) / (32ll * h.groups);
    return g;
}

template <class T, int V, int K>
int32_t ln_launch_fwd(const LnChoice& h, const LnGeom& g, const void* x, const RunStrides& xs, void* y,
                      const RunStrides& ys, const void* scale, const void* bias, float eps, void* mean, void* inv_std,
                      cudaStream_t stream)
{
    DCB_REQUIRE(g.tiles < (1ll << 31), "too many cells");
    const size_t smem = h.g > 1 ? sizeof(float) * h.groups * h.g * 2 * 32 * V : 0;
    DCB_CUDA_TRY(launch_overlapped(ln_fwd_kernel<T, V, K>, dim3((unsigned) g.tiles), 32 * h.g * h.groups, smem, stream,
                                   static_cast<const T*>(x), xs, static_cast<T*>(y), ys,
                                   static_cast<const float*>(scale), static_cast<const float*>(bias), eps,
                                   static_cast<float*>(mean), static_cast<float*>(inv_std), g));
    return DCB_OK;
}

template <class T, int V, int K>
int32_t ln_launch_bwd(const LnChoice& h, const LnGeom& g, unsigned blocks, const void* x, const RunStrides& xs,
                      const void* dy, const RunStrides& dys, const void* mean, const void* inv_std, const void* scale,
                      void* dx, const RunStrides& dxs, float* partial, cudaStream_t stream)
{
    const int warps = h.g * h.groups;
    const size_t smem = sizeof(float)
                        * std::max(h.g > 1 ? 2 * warps * 2 * 32 * V : 0, partial ? 2 * warps * K : 0);
    if (smem > 48 * 1024)
        if (int32_t e = allow_dynamic_smem((const void*) ln_bwd_kernel<T, V, K>, 160 * 1024))
            return e;
    DCB_CUDA_TRY(launch_overlapped(ln_bwd_kernel<T, V, K>, dim3(blocks), 32 * warps, smem, stream,
                                   static_cast<const T*>(x), xs, static_cast<const T*>(dy), dys,
                                   static_cast<const float*>(mean), static_cast<const float*>(inv_std),
                                   static_cast<const float*>(scale), static_cast<T*>(dx), dxs, partial, g));
    return DCB_OK;
}

// f<V, K>() for the choice.
template <class F>
int32_t ln_with_shape(const LnChoice& h, F f)
{
    using std::integral_constant;
#define DCB_LN_CASE(VV, KK)                                                                                            \
    if (h.v == VV && h.k == KK)                                                                                        \
        return f(integral_constant<int, VV>(), integral_constant<int, KK>());
    DCB_LN_CASE(4, 4)
    DCB_LN_CASE(4, 8)
    DCB_LN_CASE(2, 4)
    DCB_LN_CASE(2, 8)
    DCB_LN_CASE(2, 16)
    DCB_LN_CASE(1, 4)
    DCB_LN_CASE(1, 8)
    DCB_LN_CASE(1, 16)
    DCB_LN_CASE(1, 32)
#undef DCB_LN_CASE
    set_last_error("layer norm: no kernel for this shape");
    return DCB_UNSUPPORTED;
}

} // namespace
} // namespace dcb

using namespace dcb;

extern "C" {

int32_t dcb_ln_fwd(const dcb_nd_desc* xd, int32_t dtype, const void* x, const void* scale, const void* bias, float eps,
                   const dcb_nd_desc* yd, void* y, void* mean, void* inv_std, void* stream)
{
    if (int32_t e = ln_check(xd, dtype))
        return e;
    if (int32_t e = check_nd_desc(yd))
        return e;
    DCB_REQUIRE(same_extents(*xd, *yd), "x and y differ in extents");
    DCB_REQUIRE(eps >= 0.f, "eps must not be negative");
    if (ln_empty(xd))
        return DCB_OK;
    DCB_REQUIRE(x && y, "null tensor");
    const int level = ln_level({xd, yd});
    DCB_REQUIRE(level >= 0, "W must have unit stride");
    RunGeom rg;
    RunStrides xs, ys;
    make_runs(*xd, level, &rg, &xs);
    make_runs(*yd, level, &rg, &ys);
    drop_unused_strides(rg, &xs);
    drop_unused_strides(rg, &ys);
    const RunStrides none = {};
    const int es = elem_bytes(dtype);
    const int vmax = std::min(std::min(run_vec_of(rg, xs, x, es), run_vec_of(rg, ys, y, es)),
                              std::min(run_vec_of(rg, none, mean, 4), run_vec_of(rg, none, inv_std, 4)));
    const LnChoice h = ln_choose((int) rg.c, vmax, rg.n * rg.rows * rg.len);
    const LnGeom g = ln_geometry(rg, h);
    return ln_with_types(dtype, [&](auto t) -> int32_t {
        using T = decltype(t);
        if (h.wide)
        {
            const unsigned blocks = (unsigned) std::min<long long>(g.tiles, 4ll * num_sms());
            DCB_CUDA_TRY(launch_overlapped(ln_fwd_wide_kernel<T>, dim3(blocks), 32 * LN_WIDE_WARPS, 0,
                                           as_stream(stream), static_cast<const T*>(x), xs, static_cast<T*>(y), ys,
                                           static_cast<const float*>(scale), static_cast<const float*>(bias), eps,
                                           static_cast<float*>(mean), static_cast<float*>(inv_std), g));
            return DCB_OK;
        }
        return ln_with_shape(h, [&](auto v, auto k) {
            return ln_launch_fwd<T, decltype(v)::value, decltype(k)::value>(h, g, x, xs, y, ys, scale, bias, eps, mean,
                                                                            inv_std, as_stream(stream));
        });
    });
}

int64_t dcb_ln_bwd_workspace_bytes(const dcb_nd_desc* xd, int32_t dtype)
{
    if (ln_check(xd, dtype))
        return -1;
    return 4 * 2 * xd->c * ln_blocks_max();
}

int32_t dcb_ln_bwd(const dcb_nd_desc* xd, int32_t dtype, const void* x, const dcb_nd_desc* dyd, const void* dy,
                   const void* mean, const void* inv_std, const void* scale, const dcb_nd_desc* dxd, void* dx,
                   void* dscale, void* dbias, void* workspace, int64_t workspace_bytes, void* stream)
{
    if (int32_t e = ln_check(xd, dtype))
        return e;
    if (int32_t e = check_nd_desc(dyd))
        return e;
    if (int32_t e = check_nd_desc(dxd))
        return e;
    DCB_REQUIRE(same_extents(*xd, *dyd) && same_extents(*xd, *dxd), "x, dy and dx differ in extents");
    DCB_REQUIRE((dscale == nullptr) == (dbias == nullptr), "dscale and dbias are wanted together");
    const int c = (int) xd->c;
    cudaStream_t s = as_stream(stream);
    if (ln_empty(xd))
    {
        if (dscale)
        {
            ln_zero_kernel<<<(c + 255) / 256, 256, 0, s>>>(static_cast<float*>(dscale), static_cast<float*>(dbias), c);
            DCB_LAUNCH_CHECK();
        }
        return DCB_OK;
    }
    DCB_REQUIRE(x && dy && dx && mean && inv_std, "null tensor");
    const int level = ln_level({xd, dyd, dxd});
    DCB_REQUIRE(level >= 0, "W must have unit stride");
    if (dscale)
    {
        DCB_REQUIRE(workspace && workspace_bytes >= dcb_ln_bwd_workspace_bytes(xd, dtype), "workspace too small");
        DCB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
    }
    RunGeom rg;
    RunStrides xs, dys, dxs;
    make_runs(*xd, level, &rg, &xs);
    make_runs(*dyd, level, &rg, &dys);
    make_runs(*dxd, level, &rg, &dxs);
    drop_unused_strides(rg, &xs);
    drop_unused_strides(rg, &dys);
    drop_unused_strides(rg, &dxs);
    const RunStrides none = {};
    const int es = elem_bytes(dtype);
    int vmax = std::min(run_vec_of(rg, xs, x, es), std::min(run_vec_of(rg, dys, dy, es), run_vec_of(rg, dxs, dx, es)));
    vmax = std::min(vmax, std::min(run_vec_of(rg, none, mean, 4), run_vec_of(rg, none, inv_std, 4)));
    const LnChoice h = ln_choose(c, vmax, rg.n * rg.rows * rg.len);
    const LnGeom g = ln_geometry(rg, h);
    float* partial = dscale ? static_cast<float*>(workspace) : nullptr;
    unsigned blocks = 0;
    const int32_t e = ln_with_types(dtype, [&](auto t) -> int32_t {
        using T = decltype(t);
        if (h.wide)
        {
            blocks = (unsigned) std::min<long long>(g.tiles, num_sms());
            const int smem = 8 * c;
            if (int32_t err = allow_dynamic_smem((const void*) ln_bwd_wide_kernel<T>, 8 * LN_MAX_CHANNELS))
                return err;
            DCB_CUDA_TRY(launch_overlapped(ln_bwd_wide_kernel<T>, dim3(blocks), 32 * LN_WIDE_WARPS, smem, s,
                                           static_cast<const T*>(x), xs, static_cast<const T*>(dy), dys,
                                           static_cast<const float*>(mean), static_cast<const float*>(inv_std),
                                           static_cast<const float*>(scale), static_cast<T*>(dx), dxs, partial, g));
            return DCB_OK;
        }
        // about 16 warps an SM: what 128 registers a thread leave room for
        blocks = (unsigned) std::min<long long>(
            g.tiles, std::min<long long>(ln_blocks_max(), (long long) num_sms() * std::max(1, 16 / (h.g * h.groups))));
        return ln_with_shape(h, [&](auto v, auto k) {
            return ln_launch_bwd<T, decltype(v)::value, decltype(k)::value>(h, g, blocks, x, xs, dy, dys, mean,
                                                                            inv_std, scale, dx, dxs, partial, s);
        });
    });
    if (e != DCB_OK || !dscale)
        return e;
    DCB_CUDA_TRY(launch_overlapped(ln_fold_kernel, dim3((2 * c + 7) / 8), 256, 0, s, (const float*) partial,
                                   (int) blocks, c, static_cast<float*>(dscale), static_cast<float*>(dbias)));
    return DCB_OK;
}

} // extern "C"
