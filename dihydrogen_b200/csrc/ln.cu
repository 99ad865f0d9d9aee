// Layer normalisation over the channels of every cell, forward and backward.
//
// In NC[D]HW a cell's channels lie a volume apart, its neighbours in W beside it.  A warp's
// lanes therefore take neighbouring cells, V each, and a cell's C channels are dealt out to the G
// warps of a group: all accesses are coalesced, and what the warps of a group exchange is two
// floats a cell (their sum and their centred sum of squares forward, the two sums of the gradient
// backward).  The channels are walked over twice, eight at a time, the second time out of L1 or L2,
// where a tile of 32 V cells still is: HBM sees two tensors forward, three backward.  (With all of a
// thread's channels in registers instead, addresses and predicates of the unrolled accesses took 50
// instructions an element and 15 million bf16 values in rows of odd length 40 us.)
//
// Bound by HBM: 64 x 96^3 fp32 81 us forward, 112 backward (5.6 and 6.1 TB/s).  Rows of odd length by instruction issue:
// 2 x 200 x 19 x 37 x 53 bf16 forward 21 us (2.9 TB/s).
#include "elem.cuh"

namespace dcb
{
namespace
{

constexpr int LN_STEP = 8;    // channels at a time
constexpr int LN_WARPS = 8;   // of a block; a group has 1, 2, 4 or all of them
constexpr int LN_MAX_CHANNELS = 16384; // the backward kernel's sums of a channel fill 128 KB of shared memory

// Blocks of the backward kernel that an SM's registers hold.
__host__ __device__ constexpr int ln_bwd_blocks(int v)
{
    return v == 1 ? 4 : 2;
}

struct LnGeom
{
    CellUnits units;  // of V cells (FLAT) or of 32 V
    long long per_run, rows, rows_inner;
    int c, g;         // channels; warps of a group
    float inv_c;
    long long tiles;  // of all groups of a block
};

// How a warp's cells lie.  FLAT: units of V neighbours packed over short runs.  SPLIT: 32 V cells of one run that starts
// off the alignment of accesses of V, a lane's are 32 apart; everything but the lane is the same for a warp then, so that a
// channel's address costs no instruction of the lanes.
enum LnMode
{
    LN_FLAT,
    LN_SPLIT
};

template <int V, int MODE>
struct LnAt
{
    using Lane = std::conditional_t<MODE == LN_FLAT, long long, uint32_t>;
    CellAt cell; // the thread's first cell (FLAT), the warp's (else)
    Lane lane;   // what a thread adds to the offset of that
    int have;    // cells of the thread that are there
    bool full;   // all cells of the warp are

    __device__ __forceinline__ LnAt(const LnGeom& g, long long first, int l)
    {
        if (MODE == LN_FLAT)
        {
            const bool live = first + l < g.units.total;
            cell = cell_at<V>(g.units, g.per_run, g.rows, g.rows_inner, live ? first + l : 0);
            have = live ? V : 0;
            full = first + 32 <= g.units.total;
            lane = 0;
            return;
        }
        const long long chunk = first >> 5;
        const bool live = chunk < g.units.total;
        cell = cell_at<32 * V>(g.units, g.per_run, g.rows, g.rows_inner, live ? chunk : 0);
        const long long left = live ? g.units.len - cell.pos : 0;
        full = left >= 32 * V;
        lane = l;
        have = full ? V : l < left ? (int) (left - l + 31) / 32 : 0;
    }
    __device__ __forceinline__ long long stat(const LnGeom& g) const { return cell.n * g.units.cells + cell.cell; }
};

// Values as they are stored; converted where they are used, since a conversion right behind a load waits for it.
template <class T, int V, int MODE>
struct LnRaw
{
    RawElems<T, V> r;
    template <bool FULL>
    __device__ __forceinline__ void load(const T* p, int have)
    {
        if (FULL || have > 0)
            r.load(p);
        else
            r.clear();
    }
    __device__ __forceinline__ float get(int e) const { return r.get(e); }
};

template <class T, int V>
struct LnRaw<T, V, LN_SPLIT> : SplitElems<T, V>
{};

template <int V, int MODE, bool FULL, class T>
__device__ __forceinline__ void ln_store(T* p, const float (&v)[V], int have)
{
    if constexpr (MODE == LN_SPLIT)
        store_split<V, FULL>(p, v, have);
    else if (FULL || have > 0)
        store_elems<V>(p, v);
}

// Sum over the warps of a group of what each of them left for this thread's cells.
template <int V>
__device__ __forceinline__ void ln_gather(const float* part, int g, int lane, float (&sum)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e)
        sum[e] = 0.f;
#pragma unroll 4
    for (int i = 0; i < g; ++i)
    {
        float t[V];
        load_elems<V>(part + (i * 32 + lane) * V, t);
#pragma unroll
        for (int e = 0; e < V; ++e)
            sum[e] += t[e];
    }
}

// What a thread is in its block.
struct LnSelf
{
    int lane, groups, group, cg;
    int count; // its channels: cg, cg + g, ...
    __device__ __forceinline__ LnSelf(const LnGeom& g)
    {
        const int warp = __shfl_sync(~0u, (int) threadIdx.x >> 5, 0); // known to be uniform
        lane = threadIdx.x & 31;
        groups = LN_WARPS / g.g;
        group = warp / g.g;
        cg = warp - group * g.g;
        count = (g.c - cg + g.g - 1) / g.g;
    }
};

// The warps of a group wait for one another only: how many cells a group has, and so which code its barriers stand in, is
// its own.  Barrier 0 is the block's.
__device__ __forceinline__ void ln_group_sync(const LnGeom& g, const LnSelf& me)
{
    asm volatile("bar.sync %0, %1;" ::"r"(1 + me.group), "r"(32 * g.g) : "memory");
}

template <int M>
struct LnSome
{
    static constexpr int value = M;
};

// f(first channel, how many), eight at a time and the rest in powers of two, so that how many there are is known when
// compiled.  (Predicates on each of eight took twice the time for 50 channels.)
template <bool FULL, class F>
__device__ __forceinline__ void ln_steps(int count, F f)
{
    int i = 0;
#pragma unroll 1
    for (; i + LN_STEP <= count; i += LN_STEP)
        f(i, LnSome<LN_STEP>());
    if constexpr (FULL)
    {
        if (count & 4)
            f(i, LnSome<4>()), i += 4;
        if (count & 2)
            f(i, LnSome<2>()), i += 2;
        if (count & 1)
            f(i, LnSome<1>());
    }
    else
    {
#pragma unroll 1
        for (; i < count; ++i)
            f(i, LnSome<1>());
    }
}

template <class T, int V, int MODE, bool FULL, bool KEEP>
__device__ __forceinline__ void ln_fwd_tile(const T* x, const RunStrides& xs, T* y, const RunStrides& ys,
                                            const float* __restrict__ scale, const float* __restrict__ bias, float eps,
                                            float* mean_out, float* inv_std_out, const LnGeom& geo, const LnSelf& me,
                                            const LnAt<V, MODE>& at, float* sums, float* squares)
{
    const T* px = x + (offset_of(at.cell, xs) + me.cg * xs.sc) + at.lane;
    const long long x_step = geo.g * xs.sc;
    // Mean and centred squares of eight channels at a time, joined with those before (Chan et al.).  Every mean goes with
    // what its rounding left, `rest`: a difference of rounded means would put an error of first order in |mean| /
    // deviation into the squares (64 channels, mean 1000, deviation 1: 2.6e-5 of inv_std, so 1.7e-7).  Steps are powers
    // of two, and bf16 values whose sum is rounded at all differ by as much as they are large: only fp32 steps leave a
    // rest.
    constexpr bool ROUNDED = sizeof(T) == 4;
    float mean[V], rest[V], m2[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
        mean[e] = rest[e] = m2[e] = 0.f;
    const T* p = px;
    const auto fetch = [&](auto& v, auto some) {
#pragma unroll
        for (int k = 0; k < decltype(some)::value; ++k, p += x_step)
            v[k].template load<FULL>(p, at.have);
    };
    const auto take = [&](int i, const auto& v, auto some) {
        constexpr int m = decltype(some)::value;
        const float inv_m = 1.f / m, f = m / (float) (i + m);
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            float s = 0.f, q = 0.f, r = 0.f;
#pragma unroll
            for (int k = 0; k < m; ++k)
                s += v[k].get(e);
            s *= inv_m;
#pragma unroll
            for (int k = 0; k < m; ++k)
            {
                const float t = v[k].get(e) - s;
                if (ROUNDED)
                    r += t;
                q = fmaf(t, t, q);
            }
            if (ROUNDED)
            {
                q = fmaf(-r, r * inv_m, q); // about the true mean of the eight, s + r / m
                q = q < 0.f ? 0.f : q;
            }
            if (KEEP)
            {
                mean[e] = s, rest[e] = r * inv_m, m2[e] = q;
                continue;
            }
            const float more = fmaf(r, inv_m, -rest[e]), step = f * (s - mean[e]), d = s - mean[e] + more;
            const float joined = mean[e] + step;
            rest[e] = (mean[e] - joined + step) + fmaf(f, more, rest[e]);
            mean[e] = joined;
            m2[e] += fmaf(d * d, f * i, q);
        }
    };
    LnRaw<T, V, MODE> kept[LN_STEP];
    if (KEEP)
    {
        fetch(kept, LnSome<LN_STEP>());
        take(0, kept, LnSome<LN_STEP>());
    }
    else
        ln_steps<FULL>(me.count, [&](int i, auto some) {
            LnRaw<T, V, MODE> v[decltype(some)::value];
            fetch(v, some);
            take(i, v, some);
        });
#pragma unroll
    for (int e = 0; e < V && (ROUNDED || !KEEP); ++e)
    {
        const float whole = mean[e] + rest[e];
        rest[e] = mean[e] - whole + rest[e];
        mean[e] = whole == whole ? whole : mean[e]; // an infinite mean leaves no number behind
    }
    if (geo.g > 1)
    {
        float all[V];
#pragma unroll
        for (int e = 0; e < V; ++e)
            all[e] = mean[e] * me.count;
        store_elems<V>(sums + (me.cg * 32 + me.lane) * V, all);
        ln_group_sync(geo, me);
        ln_gather<V>(sums, geo.g, me.lane, all);
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            const float d = mean[e] - all[e] * geo.inv_c + rest[e];
            m2[e] = fmaf(d * d, (float) me.count, m2[e]);
            mean[e] = all[e] * geo.inv_c;
        }
        store_elems<V>(squares + (me.cg * 32 + me.lane) * V, m2);
        ln_group_sync(geo, me); // behind it nobody reads `sums`, and behind the next tile's first nobody `squares`
        ln_gather<V>(squares, geo.g, me.lane, m2);
    }
    float inv[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
        inv[e] = 1.f / sqrtf(fmaf(m2[e], geo.inv_c, eps));
    if (me.cg == 0)
    {
        const long long i = at.stat(geo);
        if (mean_out)
            ln_store<V, MODE, FULL>(mean_out + i + at.lane, mean, at.have);
        if (inv_std_out)
            ln_store<V, MODE, FULL>(inv_std_out + i + at.lane, inv, at.have);
    }
    p = px;
    T* py = y + (offset_of(at.cell, ys) + me.cg * ys.sc) + at.lane;
    const long long y_step = geo.g * ys.sc;
    const auto give = [&](int i, const auto& v, auto some) {
        constexpr int m = decltype(some)::value;
        float w[m], b[m];
#pragma unroll
        for (int k = 0; k < m; ++k)
        {
            const int c = me.cg + (i + k) * geo.g;
            w[k] = scale ? __ldg(scale + c) : 1.f;
            b[k] = bias ? __ldg(bias + c) : 0.f;
        }
#pragma unroll
        for (int k = 0; k < m; ++k, py += y_step)
        {
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
                out[e] = fmaf((v[k].get(e) - mean[e]) * inv[e], w[k], b[k]);
            ln_store<V, MODE, FULL>(py, out, at.have);
        }
    };
    if (KEEP)
        give(0, kept, LnSome<LN_STEP>());
    else
        ln_steps<FULL>(me.count, [&](int i, auto some) {
            LnRaw<T, V, MODE> v[decltype(some)::value];
            fetch(v, some);
            give(i, v, some);
        });
}

// Shared memory: the groups' sums and their centred sums of squares.
template <class T, int V, int MODE, bool KEEP>
__global__ void __launch_bounds__(32 * LN_WARPS, 4)
    ln_fwd_kernel(const T* x, RunStrides xs, T* y, RunStrides ys, const float* scale, const float* bias, float eps,
                  float* mean_out, float* inv_std_out, LnGeom geo)
{
    __shared__ float4 room[2 * LN_WARPS * 32 * V / 4];
    const LnSelf me(geo);
    float* sums = reinterpret_cast<float*>(room) + me.group * geo.g * 32 * V;
    float* squares = sums + LN_WARPS * 32 * V;
    wait_for_previous_kernel(x, scale, bias);
    for (long long tile = blockIdx.x; tile < geo.tiles; tile += gridDim.x)
    {
        const LnAt<V, MODE> at(geo, (tile * me.groups + me.group) * 32, me.lane);
        if (at.full)
            ln_fwd_tile<T, V, MODE, true, KEEP>(x, xs, y, ys, scale, bias, eps, mean_out, inv_std_out, geo, me, at, sums,
                                          squares);
        else
            ln_fwd_tile<T, V, MODE, false, KEEP>(x, xs, y, ys, scale, bias, eps, mean_out, inv_std_out, geo, me, at, sums,
                                           squares);
    }
    dependents_may_start();
}

template <class T, int V, int MODE, bool FULL, bool KEEP>
__device__ __forceinline__ void ln_bwd_tile(const T* x, const RunStrides& xs, const T* dy, const RunStrides& dys,
                                            const float* mean_in, const float* inv_std_in,
                                            const float* __restrict__ scale, T* dx, const RunStrides& dxs, bool grads,
                                            const LnGeom& geo, const LnSelf& me, const LnAt<V, MODE>& at, float* mine,
                                            float* acc)
{
    // what is not there is loaded as zeros and adds nothing
    LnRaw<float, V, MODE> mean, inv;
    const long long stat = at.stat(geo);
    mean.template load<FULL>(mean_in + stat + at.lane, at.have);
    inv.template load<FULL>(inv_std_in + stat + at.lane, at.have);
    const T* px = x + (offset_of(at.cell, xs) + me.cg * xs.sc) + at.lane;
    const T* pd = dy + (offset_of(at.cell, dys) + me.cg * dys.sc) + at.lane;
    const long long x_step = geo.g * xs.sc, dy_step = geo.g * dys.sc;
    float a[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e)
        a[e] = b[e] = 0.f;
    const T *p = px, *d = pd;
    const auto fetch = [&](auto& x_of, auto& dy_of, auto some) {
#pragma unroll
        for (int k = 0; k < decltype(some)::value; ++k, p += x_step, d += dy_step)
        {
            x_of[k].template load<FULL>(p, at.have);
            dy_of[k].template load<FULL>(d, at.have);
        }
    };
    const auto take = [&](int i, const auto& x_of, const auto& dy_of, auto some) {
        constexpr int m = decltype(some)::value;
        float sw[m], sb[m];
#pragma unroll
        for (int k = 0; k < m; ++k)
        {
            sw[k] = sb[k] = 0.f;
            const float w = scale ? __ldg(scale + me.cg + (i + k) * geo.g) : 1.f;
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                const float u = (x_of[k].get(e) - mean.get(e)) * inv.get(e), y = dy_of[k].get(e), g = y * w;
                sw[k] = fmaf(y, u, sw[k]);
                sb[k] += y;
                a[e] += g;
                b[e] = fmaf(g, u, b[e]);
            }
        }
        if (grads) // a channel belongs to one warp of the group
        {
            const float tw = lane_sums<m>(sw, me.lane), tb = lane_sums<m>(sb, me.lane);
            const int c = me.cg + (i + me.lane) * geo.g;
            if (me.lane < m)
            {
                acc[c] += tw;
                acc[geo.c + c] += tb;
            }
        }
    };
    LnRaw<T, V, MODE> x_kept[LN_STEP], dy_kept[LN_STEP];
    if (KEEP)
    {
        fetch(x_kept, dy_kept, LnSome<LN_STEP>());
        take(0, x_kept, dy_kept, LnSome<LN_STEP>());
    }
    else
        ln_steps<FULL>(me.count, [&](int i, auto some) {
            LnRaw<T, V, MODE> x_of[decltype(some)::value], dy_of[decltype(some)::value];
            fetch(x_of, dy_of, some);
            take(i, x_of, dy_of, some);
        });
    if (geo.g > 1)
    {
        store_elems<V>(mine + (me.cg * 32 + me.lane) * V, a);
        store_elems<V>(mine + (LN_WARPS * 32 + me.cg * 32 + me.lane) * V, b);
        ln_group_sync(geo, me); // the other half of the sums' room is free again behind the next tile's barrier
        ln_gather<V>(mine, geo.g, me.lane, a);
        ln_gather<V>(mine + LN_WARPS * 32 * V, geo.g, me.lane, b);
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        a[e] *= geo.inv_c, b[e] *= geo.inv_c;
    p = px, d = pd;
    T* po = dx + (offset_of(at.cell, dxs) + me.cg * dxs.sc) + at.lane;
    const long long dx_step = geo.g * dxs.sc;
    const auto give = [&](int i, const auto& x_of, const auto& dy_of, auto some) {
        constexpr int m = decltype(some)::value;
        float w[m];
#pragma unroll
        for (int k = 0; k < m; ++k)
            w[k] = scale ? __ldg(scale + me.cg + (i + k) * geo.g) : 1.f;
#pragma unroll
        for (int k = 0; k < m; ++k, po += dx_step)
        {
            float out[V];
#pragma unroll
            for (int e = 0; e < V; ++e)
            {
                const float u = (x_of[k].get(e) - mean.get(e)) * inv.get(e);
                out[e] = inv.get(e) * (fmaf(dy_of[k].get(e), w[k], -a[e]) - u * b[e]);
            }
            ln_store<V, MODE, FULL>(po, out, at.have);
        }
    };
    if (KEEP)
        give(0, x_kept, dy_kept, LnSome<LN_STEP>());
    else
        ln_steps<FULL>(me.count, [&](int i, auto some) {
            LnRaw<T, V, MODE> x_of[decltype(some)::value], dy_of[decltype(some)::value];
            fetch(x_of, dy_of, some);
            give(i, x_of, dy_of, some);
        });
}

// Blocks walk over the tiles.  The gradients of scale and bias are added up over a tile's cells by exchanges between
// the lanes, over the tiles in shared memory, [group][2][c], and leave as partial[which][channel][block].
template <class T, int V, int MODE, bool KEEP>
__global__ void __launch_bounds__(32 * LN_WARPS, ln_bwd_blocks(V))
    ln_bwd_kernel(const T* x, RunStrides xs, const T* dy, RunStrides dys, const float* mean_in,
                  const float* inv_std_in, const float* scale, T* dx, RunStrides dxs, float* partial, LnGeom geo)
{
    extern __shared__ float acc[];
    __shared__ float4 room[2][2 * LN_WARPS * 32 * V / 4];
    const LnSelf me(geo);
    if (partial)
        for (int i = threadIdx.x; i < 2 * geo.c * me.groups; i += 32 * LN_WARPS)
            acc[i] = 0.f;
    wait_for_previous_kernel(x, dy, mean_in, inv_std_in, scale);
    __syncthreads();
    int turn = 0;
    for (long long tile = blockIdx.x; tile < geo.tiles; tile += gridDim.x, turn ^= 1)
    {
        const LnAt<V, MODE> at(geo, (tile * me.groups + me.group) * 32, me.lane);
        float* mine = reinterpret_cast<float*>(room[turn]) + me.group * geo.g * 32 * V;
        float* sums = acc + me.group * 2 * geo.c;
        if (at.full)
            ln_bwd_tile<T, V, MODE, true, KEEP>(x, xs, dy, dys, mean_in, inv_std_in, scale, dx, dxs, partial != nullptr, geo,
                                          me, at, mine, sums);
        else
            ln_bwd_tile<T, V, MODE, false, KEEP>(x, xs, dy, dys, mean_in, inv_std_in, scale, dx, dxs, partial != nullptr,
                                           geo, me, at, mine, sums);
    }
    dependents_may_start();
    if (!partial)
        return;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * geo.c; i += 32 * LN_WARPS)
    {
        float s = 0.f;
        for (int p = 0; p < me.groups; ++p)
            s += acc[p * 2 * geo.c + i];
        partial[(long long) i * gridDim.x + blockIdx.x] = s;
    }
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

// What a launch is made of: cells of a thread, warps of a group, how the cells lie.
struct LnChoice
{
    int v, g, mode;
    bool keep; // every thread has eight channels: they stay in registers
};

// vmax: neighbours that one access may fetch.  len: cells of a run.
LnChoice ln_choose(int c, int vmax, long long len, long long cells)
{
    LnChoice h;
    // Four cells a thread where that leaves every SM a block of tiles (64 x 96^3 fp32, forward and backward, 81 + 112 us,
    // 136 + 160 with one; 32 x 2 x 64^2, 4.5 + 4.5 and 3.9 + 4.5 with one), 32 apart where accesses of four are not aligned
    // (200 x 2 x 19 x 37 x 53 bf16 17 + 31 us, with one 29 + 55) and runs are so long that their last tiles waste a quarter
    // of the lanes at most.
    const bool four = cells >= 4ll * 32 * num_sms();
    h.mode = four && vmax < 4 && len >= 512 ? LN_SPLIT : LN_FLAT;
    h.v = h.mode == LN_SPLIT || (four && vmax == 4) ? 4 : 1;
    // as many warps a group as have eight channels each, more where there are few tiles
    const long long tiles = (cells + 32 * h.v - 1) / (32 * h.v);
    h.g = 1;
    while (h.g < LN_WARPS && (c > LN_STEP * h.g || (c >= 2 * h.g && tiles * h.g < 8ll * num_sms())))
        h.g *= 2;
    h.keep = c == LN_STEP * h.g; // (64 x 96^3 fp32 87 + 131 us without)
    return h;
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
    g.per_run = h.mode == LN_FLAT ? rg.len / h.v : (rg.len + 32 * h.v - 1) / (32 * h.v);
    g.units = cell_units_of(rg, g.per_run);
    g.rows = rg.rows;
    g.rows_inner = rg.rows_inner;
    g.c = (int) rg.c;
    g.g = h.g;
    g.inv_c = 1.f / g.c;
    const long long a_tile = LN_WARPS / h.g * (h.mode == LN_FLAT ? 32 : 1); // units
    g.tiles = (g.units.total + a_tile - 1) / a_tile;
    return g;
}

template <class T, int V, int MODE, bool KEEP>
int32_t ln_launch_fwd(const LnGeom& g, const void* x, const RunStrides& xs, void* y, const RunStrides& ys,
                      const void* scale, const void* bias, float eps, void* mean, void* inv_std, cudaStream_t stream)
{
    const unsigned blocks = (unsigned) std::min<long long>(g.tiles, 4ll * num_sms());
    DCB_CUDA_TRY(launch_overlapped(ln_fwd_kernel<T, V, MODE, KEEP>, dim3(blocks), 32 * LN_WARPS, 0, stream,
                                   static_cast<const T*>(x), xs, static_cast<T*>(y), ys,
                                   static_cast<const float*>(scale), static_cast<const float*>(bias), eps,
                                   static_cast<float*>(mean), static_cast<float*>(inv_std), g));
    return DCB_OK;
}

template <class T, int V, int MODE, bool KEEP>
int32_t ln_launch_bwd(const LnGeom& g, unsigned blocks, const void* x, const RunStrides& xs, const void* dy,
                      const RunStrides& dys, const void* mean, const void* inv_std, const void* scale, void* dx,
                      const RunStrides& dxs, float* partial, cudaStream_t stream)
{
    const int smem = partial ? 8 * g.c * (LN_WARPS / g.g) : 0;
    if (smem > 32 * 1024)
        if (int32_t e = allow_dynamic_smem((const void*) ln_bwd_kernel<T, V, MODE, KEEP>, 8 * LN_MAX_CHANNELS))
            return e;
    DCB_CUDA_TRY(launch_overlapped(ln_bwd_kernel<T, V, MODE, KEEP>, dim3(blocks), 32 * LN_WARPS, smem, stream,
                                   static_cast<const T*>(x), xs, static_cast<const T*>(dy), dys,
                                   static_cast<const float*>(mean), static_cast<const float*>(inv_std),
                                   static_cast<const float*>(scale), static_cast<T*>(dx), dxs, partial, g));
    return DCB_OK;
}

// f(V, MODE, KEEP) for the choice.
template <class F>
int32_t ln_with_shape(const LnChoice& h, F f)
{
    using std::integral_constant;
    const auto shape = [&](auto keep) -> int32_t {
        if (h.mode == LN_SPLIT)
            return f(integral_constant<int, 4>(), integral_constant<int, LN_SPLIT>(), keep);
        return h.v == 4 ? f(integral_constant<int, 4>(), integral_constant<int, LN_FLAT>(), keep)
                        : f(integral_constant<int, 1>(), integral_constant<int, LN_FLAT>(), keep);
    };
    return h.keep ? shape(std::bool_constant<true>()) : shape(std::bool_constant<false>());
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
    DCB_REQUIRE(x != y || same_strides(*xd, *yd), "in place the strides must be the same");
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
    const LnChoice h = ln_choose((int) rg.c, vmax, rg.len, rg.n * rg.rows * rg.len);
    const LnGeom g = ln_geometry(rg, h);
    return ln_with_types(dtype, [&](auto t) -> int32_t {
        using T = decltype(t);
        return ln_with_shape(h, [&](auto v, auto mode, auto keep) {
            return ln_launch_fwd<T, decltype(v)::value, decltype(mode)::value, decltype(keep)::value>(
                g, x, xs, y, ys, scale, bias, eps, mean, inv_std, as_stream(stream));
        });
    });
}

int64_t dcb_ln_bwd_workspace_bytes(const dcb_nd_desc* xd, int32_t dtype)
{
    if (ln_check(xd, dtype))
        return -1;
    return 4 * 2 * xd->c * ln_bwd_blocks(1) * (int64_t) num_sms();
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
    DCB_REQUIRE((dx != x || same_strides(*dxd, *xd)) && (dx != dy || same_strides(*dxd, *dyd)),
                "in place the strides must be the same");
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
    const LnChoice h = ln_choose(c, vmax, rg.len, rg.n * rg.rows * rg.len);
    const LnGeom g = ln_geometry(rg, h);
    float* partial = dscale ? static_cast<float*>(workspace) : nullptr;
    const unsigned blocks = (unsigned) std::min<long long>(g.tiles, (long long) ln_bwd_blocks(h.v) * num_sms());
    const int32_t e = ln_with_types(dtype, [&](auto t) -> int32_t {
        using T = decltype(t);
        return ln_with_shape(h, [&](auto v, auto mode, auto keep) {
            return ln_launch_bwd<T, decltype(v)::value, decltype(mode)::value, decltype(keep)::value>(
                g, blocks, x, xs, dy, dys, mean,
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
