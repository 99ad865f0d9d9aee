// Rotary positions on a grid: pairs of a head's channels turned by angles that grow along D, H
// and W.
//
// One pass over the tensor, HBM bound.  The angles depend on a pair and on one coordinate of a
// cell, not on the sample or the head: a thread owns a pair of channels at V neighbouring cells,
// looks up V cosines and sines in the plan's tables (a few hundred kilobytes, in L2) and walks
// over the heads with them, several heads' loads in flight.  A channel of no axis is a pair with
// nothing to turn.  2 x 12 heads of 128 channels on 40^3 cells, bf16: 123 us (6.4 TB/s).
#include "elem.cuh"

#include <cmath>
#include <new>

struct dcb_rotary_plan
{
    dcb_rotary_desc rd;
    int64_t c, dims[3];
    float* tables;        // per axis: cosines [pair][position], then sines
    long long table_at[3]; // in floats
    int device;
};

namespace dcb
{
namespace
{

constexpr int ROT_HEADS = 4; // in flight a thread

struct RotArgs
{
    CellUnits units;   // of one sample
    long long per_run, rows, rows_inner;
    FastDiv w, h;      // a cell's coordinates
    const float* tables;
    long long table_at[3];
    int dims[3];       // D, H, W
    int first[3];      // an axis' first channel
    int pairs[3];      // its pairs
    int turned_pairs;  // of a head, all axes
    int head_dim, heads, rotated, interleaved;
    int head_chunks, chunk; // heads of a block: `chunk` from blockIdx.z % head_chunks on
    int skip_copies;   // in place: what is not turned is there already
    float sign;
};

template <class T, int V, bool SPLIT>
struct RotRaw
{
    RawElems<T, V> r;
    template <bool FULL>
    __device__ __forceinline__ void load(const T* p, int)
    {
        r.load(p);
    }
    __device__ __forceinline__ float get(int e) const { return r.get(e); }
};

template <class T, int V>
struct RotRaw<T, V, true> : SplitElems<T, V>
{};

// Slots of a head: its turned pairs, then the channels of no axis two at a time (the last may be alone).  A thread has V
// neighbours (units), or, SPLIT, V cells 32 apart of its warp's 32 V (units are a warp's).
template <class TX, class TY, int V, bool SPLIT>
__global__ void __launch_bounds__(256) rotary_kernel(const TX* x, RunStrides xs, TY* y, RunStrides ys, RotArgs a)
{
    wait_for_previous_kernel(x);
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const long long unit = SPLIT ? (long long) blockIdx.x * 8 + __shfl_sync(~0u, (int) threadIdx.x >> 5, 0)
                                 : (long long) blockIdx.x * 256 + threadIdx.x;
    if (unit >= a.units.total)
        return;
    const int slot = blockIdx.y;
    const long long n = blockIdx.z / a.head_chunks;
    const int head0 = (int) (blockIdx.z - n * a.head_chunks) * a.chunk;
    const int head1 = min(head0 + a.chunk, a.heads);
    CellAt at = cell_at<SPLIT ? 32 * V : V>(a.units, a.per_run, a.rows, a.rows_inner, unit);
    at.n = n;
    int have = V;
    if (SPLIT)
    {
        const long long left = a.units.len - at.pos - lane;
        have = left <= 0 ? 0 : (int) min((long long) V, (left + 31) / 32);
        at.cell += lane;
    }
    const bool full = !SPLIT || at.pos + 32 * V <= a.units.len;
    const int lane_at = SPLIT ? lane : 0;

    int c0, c1;
    float co[V], si[V];
    const bool turns = slot < a.turned_pairs;
    if (turns)
    {
        int axis = 0, j = slot;
        while (j >= a.pairs[axis])
            j -= a.pairs[axis++];
        c0 = a.first[axis] + (a.interleaved ? 2 * j : j);
        c1 = c0 + (a.interleaved ? 1 : a.pairs[axis]);
        const int len = a.dims[axis];
        const float* cos_of = a.tables + a.table_at[axis] + (long long) j * len;
        const float* sin_of = cos_of + (long long) a.pairs[axis] * len;
#pragma unroll
        for (int e = 0; e < V; ++e)
        {
            const uint32_t cell = (uint32_t) at.cell + (SPLIT ? 32 * min(e, have - 1) : e);
            const uint32_t row = a.w.div(cell), plane = a.h.div(row);
            const uint32_t p = axis == 2 ? cell - row * a.w.d : axis == 1 ? row - plane * a.h.d : plane;
            co[e] = cos_of[p];
            si[e] = a.sign * sin_of[p];
        }
    }
    else
    {
        c0 = 2 * slot; // 2 turned_pairs channels lie before
        c1 = c0 + 1 < a.head_dim ? c0 + 1 : -1;
    }

    // heads [lo, hi), several at a time: a whole group's loads go out before anything waits for one
    const TX* px = x + offset_of(at, xs) + lane_at;
    TY* py = y + offset_of(at, ys) + lane_at;
    const long long x_head = a.head_dim * xs.sc, y_head = a.head_dim * ys.sc;
    const auto heads = [&](int lo, int hi, auto turn, auto pair, auto whole) {
        constexpr bool TURN = decltype(turn)::value, PAIR = decltype(pair)::value, FULL = decltype(whole)::value;
        const auto put = [&](TY* to, const float (&v)[V]) {
            if constexpr (SPLIT)
                store_split<V, FULL>(to, v, have);
            else
                store_elems<V>(to, v);
        };
        const auto some = [&](int h, auto count) {
            constexpr int N = decltype(count)::value;
            RotRaw<TX, V, SPLIT> rp[N], rq[N];
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                rp[i].template load<FULL>(px + (h + i) * x_head + c0 * xs.sc, have);
                if (PAIR)
                    rq[i].template load<FULL>(px + (h + i) * x_head + c1 * xs.sc, have);
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
            {
                float p[V], q[V];
#pragma unroll
                for (int e = 0; e < V; ++e)
                {
                    p[e] = rp[i].get(e);
                    if (PAIR)
                        q[e] = rq[i].get(e);
                    if (TURN)
                    {
                        const float r = p[e] * co[e] - q[e] * si[e];
                        q[e] = p[e] * si[e] + q[e] * co[e];
                        p[e] = r;
                    }
                }
                put(py + (h + i) * y_head + c0 * ys.sc, p);
                if (PAIR)
                    put(py + (h + i) * y_head + c1 * ys.sc, q);
            }
        };
        int h = lo;
#pragma unroll 1
        for (; h + ROT_HEADS <= hi; h += ROT_HEADS)
            some(h, std::integral_constant<int, ROT_HEADS>());
        if (h + 2 <= hi)
            some(h, std::integral_constant<int, 2>()), h += 2;
        if (h < hi)
            some(h, std::integral_constant<int, 1>());
    };
    using std::bool_constant;
    const int turned = turns ? max(head0, min(head1, a.rotated)) : head0; // heads before are turned
    const auto all = [&](auto whole) {
        if (turns)
            heads(head0, turned, bool_constant<true>(), bool_constant<true>(), whole);
        if (a.skip_copies)
            return;
        if (c1 >= 0)
            heads(turned, head1, bool_constant<false>(), bool_constant<true>(), whole);
        else
            heads(turned, head1, bool_constant<false>(), bool_constant<false>(), whole);
    };
    if (!SPLIT || full)
        all(bool_constant<true>());
    else if (have > 0)
        all(bool_constant<false>());
}

template <class TX, class TY>
int32_t rotary_launch(int v, bool split, dim3 grid, const void* x, const RunStrides& xs, void* y, const RunStrides& ys,
                      const RotArgs& a, cudaStream_t stream)
{
    const auto go = [&](auto kernel) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(kernel, grid, 256, 0, stream, static_cast<const TX*>(x), xs,
                                       static_cast<TY*>(y), ys, a));
        return DCB_OK;
    };
    if (split)
        return go(rotary_kernel<TX, TY, 4, true>);
    if constexpr (sizeof(TX) == 2 || sizeof(TY) == 2)
        if (v == 8)
            return go(rotary_kernel<TX, TY, 8, false>);
    return v == 4 ? go(rotary_kernel<TX, TY, 4, false>) : go(rotary_kernel<TX, TY, 1, false>);
}

} // namespace
} // namespace dcb

using namespace dcb;

extern "C" {

int32_t dcb_rotary_plan_create(const dcb_rotary_desc* rd, const dcb_nd_desc* xd, dcb_rotary_plan** plan)
{
    DCB_REQUIRE(rd && plan, "null argument");
    *plan = nullptr;
    if (int32_t e = check_nd_desc(xd))
        return e;
    DCB_REQUIRE(rd->nsd == xd->nsd, "nsd differs from the tensor's");
    DCB_REQUIRE(rd->head_dim >= 1 && xd->c >= 1 && xd->c % rd->head_dim == 0 && xd->c < (1 << 30),
                "channels must be heads of head_dim");
    for (int i = 0; i < 3; ++i)
        if (xd->dims[i] >= (1ll << 31))
        {
            set_last_error("unsupported: 2^31 cells along an axis");
            return DCB_UNSUPPORTED;
        }
    const int64_t heads = xd->c / rd->head_dim;
    DCB_REQUIRE(rd->rotated_heads >= 0 && rd->rotated_heads <= heads, "rotated_heads out of range");
    int64_t turned = 0;
    long long floats = 0;
    for (int i = 0; i < 3; ++i)
    {
        DCB_REQUIRE(rd->axis_channels[i] >= 0 && rd->axis_channels[i] % 2 == 0, "axis_channels must be even");
        DCB_REQUIRE(std::isfinite(rd->step[i]), "step must be finite");
        turned += rd->axis_channels[i];
        floats += (long long) rd->axis_channels[i] * xd->dims[i];
    }
    DCB_REQUIRE(rd->nsd == 3 || rd->axis_channels[0] == 0, "a 2-D tensor has no D");
    DCB_REQUIRE(turned <= rd->head_dim, "axis_channels exceed head_dim");
    DCB_REQUIRE(std::isfinite(rd->base) && rd->base > 0, "base must be positive");
    if ((rd->head_dim + 1) / 2 > 65535 || xd->dims[0] * xd->dims[1] >= (1ll << 31) / (xd->dims[2] > 0 ? xd->dims[2] : 1))
    {
        set_last_error("unsupported: 2^31 cells of a sample, or heads of 2^17 channels");
        return DCB_UNSUPPORTED;
    }
    dcb_rotary_plan* p = new (std::nothrow) dcb_rotary_plan();
    std::vector<float> host;
    try
    {
        if (!p)
            throw std::bad_alloc();
        host.resize((size_t) floats);
    }
    catch (const std::bad_alloc&)
    {
        delete p;
        set_last_error("out of host memory");
        return DCB_BAD_ARG;
    }
    p->rd = *rd;
    p->c = xd->c;
    p->tables = nullptr;
    long long at = 0;
    for (int i = 0; i < 3; ++i)
    {
        p->dims[i] = xd->dims[i];
        p->table_at[i] = at;
        const int pairs = rd->axis_channels[i] / 2;
        // the largest angle is one end's, of the first or the last pair
        for (int j : {0, pairs - 1})
            for (double end : {(double) rd->origin[i], (double) rd->origin[i] + xd->dims[i]})
                if (pairs > 0 && !std::isfinite(rd->step[i] * end * std::pow(rd->base, -2.0 * j / rd->axis_channels[i])))
                {
                    delete p;
                    set_last_error("bad argument: positions whose angles are not finite");
                    return DCB_BAD_ARG;
                }
        for (int j = 0; j < pairs; ++j)
        {
            const double per = std::pow(rd->base, -2.0 * j / rd->axis_channels[i]);
            for (int64_t k = 0; k < xd->dims[i]; ++k)
            {
                const double angle = rd->step[i] * (double) (rd->origin[i] + k) * per;
                host[at + j * xd->dims[i] + k] = (float) std::cos(angle);
                host[at + (pairs + j) * xd->dims[i] + k] = (float) std::sin(angle);
            }
        }
        at += 2ll * pairs * xd->dims[i];
    }
    cudaError_t err = cudaGetDevice(&p->device);
    if (err == cudaSuccess && floats > 0)
    {
        err = cudaMalloc(&p->tables, floats * sizeof(float));
        if (err == cudaSuccess)
            err = cudaMemcpy(p->tables, host.data(), floats * sizeof(float), cudaMemcpyHostToDevice);
        // a copy from pageable memory returns when its source may go; kernels on other streams need it arrived
        if (err == cudaSuccess)
            err = cudaStreamSynchronize(nullptr);
    }
    if (err != cudaSuccess)
    {
        set_last_error(std::string("rotary plan: ") + cudaGetErrorString(err));
        (void) cudaGetLastError();
        if (p->tables)
            cudaFree(p->tables);
        delete p;
        return DCB_CUDA_ERROR;
    }
    *plan = p;
    return DCB_OK;
}

int32_t dcb_rotary_plan_destroy(dcb_rotary_plan* plan)
{
    if (plan)
    {
        if (plan->tables)
            cudaFree(plan->tables);
        delete plan;
    }
    return DCB_OK;
}

int32_t dcb_rotary_apply(const dcb_rotary_plan* plan, const dcb_nd_desc* xd, int32_t x_dtype, const void* x,
                         const dcb_nd_desc* yd, int32_t y_dtype, void* y, int32_t inverse, void* stream)
{
    DCB_REQUIRE(plan, "null plan");
    if (int32_t e = check_nd_desc(xd))
        return e;
    if (int32_t e = check_nd_desc(yd))
        return e;
    DCB_REQUIRE(same_extents(*xd, *yd), "x and y differ in extents");
    DCB_REQUIRE(xd->nsd == plan->rd.nsd && xd->c == plan->c && xd->dims[0] == plan->dims[0]
                    && xd->dims[1] == plan->dims[1] && xd->dims[2] == plan->dims[2],
                "extents differ from the plan's");
    DCB_REQUIRE(known_dtype(x_dtype) && known_dtype(y_dtype), "dtype must be DCB_F32 or DCB_BF16");
    if (xd->n == 0 || xd->dims[0] == 0 || xd->dims[1] == 0 || xd->dims[2] == 0)
        return DCB_OK;
    DCB_REQUIRE(x && y, "null tensor");
    DCB_REQUIRE(x != y || (x_dtype == y_dtype && same_strides(*xd, *yd)),
                "in place the types and strides must be the same");
    int device = 0;
    DCB_CUDA_TRY(cudaGetDevice(&device));
    DCB_REQUIRE(device == plan->device, "the plan lives on another device");
    const int level = std::min(run_level(*xd), run_level(*yd));
    DCB_REQUIRE(level >= 0, "W must have unit stride");
    RunGeom rg;
    RunStrides xs, ys;
    make_runs(*xd, level, &rg, &xs);
    make_runs(*yd, level, &rg, &ys);
    drop_unused_strides(rg, &xs);
    drop_unused_strides(rg, &ys);
    const int most = x_dtype == DCB_BF16 || y_dtype == DCB_BF16 ? 8 : 4; // accesses of 16 bytes
    int v = std::min(run_vec_of(rg, xs, x, elem_bytes(x_dtype), most), run_vec_of(rg, ys, y, elem_bytes(y_dtype), most));
    const dcb_rotary_desc& rd = plan->rd;
    // Eight cells a thread (16 bytes of bf16) where that leaves 16 blocks for every SM; four, or four 32 apart where
    // accesses of four are not aligned and runs are long enough that their last 128 cells are no waste; else one.
    // (2 x 1536 x 40^3 in bf16 with four cells 190 us, with eight 129; 8192 x 1536 values 8.2 and 9.5.)
    const long long heads_at_once = (xd->c / rd.head_dim + ROT_HEADS - 1) / ROT_HEADS;
    const long long pairs = (rd.head_dim + 1) / 2;
    if (v == 8 && rg.rows * rg.len / 8 / 256 * pairs * xd->n * heads_at_once < 16ll * num_sms())
        v = 4;
    const bool split = v < 4 && rg.len >= 512;
    v = split ? 4 : v < 4 ? 1 : v;
    RotArgs a = {};
    RunGeom one = rg;
    one.n = 1;
    a.per_run = split ? (rg.len + 127) / 128 : rg.len / v;
    a.units = cell_units_of(one, a.per_run);
    a.rows = rg.rows;
    a.rows_inner = rg.rows_inner;
    a.w = FastDiv::of((uint32_t) xd->dims[2]);
    a.h = FastDiv::of((uint32_t) xd->dims[1]);
    a.tables = plan->tables;
    int channel = 0;
    for (int i = 0; i < 3; ++i)
    {
        a.table_at[i] = plan->table_at[i];
        a.dims[i] = (int) xd->dims[i];
        a.first[i] = channel;
        a.pairs[i] = rd.axis_channels[i] / 2;
        channel += rd.axis_channels[i];
        a.turned_pairs += a.pairs[i];
    }
    a.head_dim = rd.head_dim;
    a.heads = (int) (xd->c / rd.head_dim);
    a.rotated = rd.rotated_heads;
    a.interleaved = rd.interleaved != 0;
    a.skip_copies = x == y;
    a.sign = inverse ? -1.f : 1.f;
    if (a.skip_copies && (a.rotated == 0 || a.turned_pairs == 0))
        return DCB_OK;
    const long long blocks_x = split ? (a.units.total + 7) / 8 : (a.units.total + 255) / 256;
    const int slots = a.turned_pairs + (rd.head_dim - channel + 1) / 2;
    // a thread keeps its angles for as many heads as leave four blocks for every SM's eight
    a.chunk = a.heads;
    while (a.chunk > ROT_HEADS
           && blocks_x * slots * xd->n * ((a.heads + a.chunk - 1) / a.chunk) < 16ll * num_sms())
        a.chunk = std::max(ROT_HEADS, a.chunk / 2);
    a.head_chunks = (a.heads + a.chunk - 1) / a.chunk;
    if (blocks_x >= (1ll << 31) || xd->n * a.head_chunks > 65535)
    {
        set_last_error("unsupported: more than 65535 samples times head groups");
        return DCB_UNSUPPORTED;
    }
    const dim3 grid((unsigned) blocks_x, slots, (unsigned) (xd->n * a.head_chunks));
    cudaStream_t s = as_stream(stream);
    if (x_dtype == DCB_F32)
        return y_dtype == DCB_F32 ? rotary_launch<float, float>(v, split, grid, x, xs, y, ys, a, s)
                                  : rotary_launch<float, bf16>(v, split, grid, x, xs, y, ys, a, s);
    return y_dtype == DCB_F32 ? rotary_launch<bf16, float>(v, split, grid, x, xs, y, ys, a, s)
                              : rotary_launch<bf16, bf16>(v, split, grid, x, xs, y, ys, a, s);
}

} // extern "C"
