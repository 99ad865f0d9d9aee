// Attention between cells: argument checks, workspace, the kernels beside the products.
#include "attention.cuh"

#include <cmath>
#include <initializer_list>
#include <utility>

namespace dcb
{
namespace
{

constexpr int ATTN_INDEX_THREADS = 1024, ATTN_INDEX_CELLS = 8; // cells of a thread at a time
constexpr int ATTN_INDEX_PARTS = 64;                             // blocks of a sample and side, at most

// Bytes of a word that are not zero.
__device__ __forceinline__ int attn_marks(uint32_t x)
{
    return __popc((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u);
}

// What a mask leaves of a sample's cells, in order.  A block has a part of a sample's cells and counts those before it by
// itself, 16 bytes of the mask at a time: 2 samples of 31 x 33 x 31 cells take 10 us; a block a sample, which went
// through them 8192 at a time, took 29.
__global__ void __launch_bounds__(ATTN_INDEX_THREADS) attn_index_kernel(const __grid_constant__ AttnProblem p)
{
    __shared__ int of_warp[32];
    __shared__ int all;
    const uint8_t* mask = blockIdx.y ? p.kv_mask : p.q_mask;
    const AttnSide side = blockIdx.y ? p.kv_side : p.q_side;
    const int cells = blockIdx.y ? p.sk : p.sq;
    constexpr long long STEP = ATTN_INDEX_THREADS * ATTN_INDEX_CELLS;
    const long long steps = (cells + STEP - 1) / STEP, part = (steps + gridDim.z - 1) / gridDim.z * STEP;
    const long long lo = blockIdx.z * part, hi = min(lo + part, (long long) cells);
    if (!mask || (lo >= cells && blockIdx.z > 0))
        return;
    wait_for_previous_kernel(mask);
    dependents_may_start();
    const long long n = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    mask += n * cells;
    int* index = side.index + n * cells;
    int* before = side.before + n * (cells + 1ll);
    int base = 0;
    if (lo > 0)
    {
        // bytes up to the first address that 16 divides, words, bytes
        const int head = (int) (-reinterpret_cast<uintptr_t>(mask) & 15);
        const uint4* words = reinterpret_cast<const uint4*>(mask + head);
        const int count = (int) ((lo - head) / 16);
        int found = 0;
#pragma unroll 4
        for (int i = threadIdx.x; i < count; i += ATTN_INDEX_THREADS)
        {
            const uint4 w = words[i];
            found += attn_marks(w.x) + attn_marks(w.y) + attn_marks(w.z) + attn_marks(w.w);
        }
        if (threadIdx.x < head)
            found += mask[threadIdx.x] != 0;
        const long long tail = head + 16ll * count + threadIdx.x;
        if (tail < lo)
            found += mask[tail] != 0;
        found = __reduce_add_sync(~0u, found);
        if (lane == 0)
            of_warp[warp] = found;
        __syncthreads();
        base = __reduce_add_sync(~0u, of_warp[lane]);
        __syncthreads();
    }
    for (long long c0 = lo; c0 < hi; c0 += STEP)
    {
        const long long i0 = c0 + threadIdx.x * ATTN_INDEX_CELLS;
        uint32_t bits = 0;
        uint8_t m[ATTN_INDEX_CELLS];
#pragma unroll
        for (int e = 0; e < ATTN_INDEX_CELLS; ++e)
            m[e] = i0 + e < cells ? mask[i0 + e] : (uint8_t) 0;
#pragma unroll
        for (int e = 0; e < ATTN_INDEX_CELLS; ++e)
            bits |= (m[e] ? 1u : 0u) << e;
        const int mine = __popc(bits);
        int sum = mine; // of this lane and those before
        for (int h = 1; h < 32; h *= 2)
        {
            const int other = __shfl_up_sync(~0u, sum, h);
            sum += lane >= h ? other : 0;
        }
        if (lane == 31)
            of_warp[warp] = sum;
        __syncthreads();
        if (warp == 0)
        {
            int w = of_warp[lane];
            for (int h = 1; h < 32; h *= 2)
            {
                const int other = __shfl_up_sync(~0u, w, h);
                w += lane >= h ? other : 0;
            }
            of_warp[lane] = w;
            if (lane == 31)
                all = w;
        }
        __syncthreads();
        int at = base + sum - mine + (warp > 0 ? of_warp[warp - 1] : 0);
        for (int e = 0; e < ATTN_INDEX_CELLS; ++e)
            if (i0 + e < cells)
            {
                before[i0 + e] = at;
                if (bits >> e & 1)
                    index[at++] = (int) (i0 + e);
            }
        base += all;
        __syncthreads();
    }
    if (threadIdx.x == 0 && hi == cells)
    {
        before[cells] = base;
        side.count[n] = base;
    }
}

// Zeros (and lse = -infinity) in the cells that a mask takes out of a result.
struct AttnZeros
{
    AttnTensor t;
    const uint8_t* mask;
    long long rows; // of a sample
    int cells;
    float* lse;     // with as many rows as heads; null
    int heads;
};

constexpr int ATTN_ZERO_ROWS = 16; // that a thread writes for one look at the mask

struct AttnZeroJobs
{
    AttnZeros job[3];
    int n;
};

template <class T>
__global__ void __launch_bounds__(256) attn_zero_kernel(const __grid_constant__ AttnZeroJobs a)
{
    const AttnZeros& z = a.job[blockIdx.y];
    const uint8_t* mask = z.mask;
    wait_for_previous_kernel(mask);
    dependents_may_start();
    const int chunks = (z.cells + 255) / 256;
    const long long rows = z.rows + z.heads; // of a sample: the tensor's, then lse's
    const long long groups = (rows + ATTN_ZERO_ROWS - 1) / ATTN_ZERO_ROWS;
    for (long long u = blockIdx.x; u < a.n * groups * chunks; u += gridDim.x)
    {
        const long long m = u / chunks, n = m / groups, row0 = (m - n * groups) * ATTN_ZERO_ROWS;
        const int i = (int) (u - m * chunks) * 256 + threadIdx.x;
        if (i >= z.cells || mask[n * z.cells + i])
            continue;
        T* to = static_cast<T*>(z.t.p) + n * z.t.sn + i;
        const float v[1] = {0.f};
#pragma unroll 4
        for (long long row = row0; row < row0 + ATTN_ZERO_ROWS; ++row)
            if (row < z.rows)
                store_elems<1>(to + row * z.t.sc, v);
            else if (row < rows)
                z.lse[(n * z.heads + row - z.rows) * z.cells + i] = -INFINITY;
    }
}

// Joins the parts of a split axis of keys: o = sum_s part_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).
template <class T>
__global__ void __launch_bounds__(256) attn_join_fwd_kernel(AttnProblem p)
{
    wait_for_previous_kernel(p.part_o, p.part_ml);
    const long long heads = (long long) p.n * p.q_heads, total = heads * p.d * p.sq;
    for (long long at = (long long) blockIdx.x * 256 + threadIdx.x; at < total; at += (long long) gridDim.x * 256)
    {
        const long long row = at / p.sq, nh = row / p.d, n = nh / p.q_heads;
        const int i = (int) (at - row * p.sq), c = (int) (row - nh * p.d);
        const float* ml = p.part_ml + nh * p.sq + i;
        const long long step = 2 * heads * p.sq;
        const bool gone = p.q_mask && !p.q_mask[n * p.sq + i]; // its parts were not written
        float m = -INFINITY;
        for (int s = 0; s < p.kv_splits && !gone; ++s)
            m = fmaxf(m, ml[s * step]);
        // a part whose only keys are NaN has no maximum, but a sum that is NaN
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f, o = 0.f;
        for (int s = 0; s < p.kv_splits && !gone; ++s)
        {
            const float f = exp2f(ml[s * step] - base);
            l = fmaf(ml[s * step + heads * p.sq], f, l);
            o = fmaf(p.part_o[s * total + at], f, o);
        }
        const bool none = l == 0.f;
        const float v[1] = {none ? 0.f : o / l};
        store_elems<1>(static_cast<T*>(p.o.p) + n * p.o.sn + ((nh - n * p.q_heads) * p.d + c) * p.o.sc + i, v);
        if (c == 0)
            p.lse[nh * p.sq + i] = none ? -INFINITY : (m + log2f(l)) / ATTN_LOG2E;
    }
}

// Adds up the parts of a gradient in order: a block a row of cells, or a piece of one.
constexpr int ATTN_JOIN_CELLS = 1024; // of a block: four a thread, 256 apart

template <class T>
__global__ void __launch_bounds__(256) attn_join_grad_kernel(const float* part, int splits, AttnTensor t, int n,
                                                             int heads, int d, int cells, const uint8_t* mask)
{
    wait_for_previous_kernel(part, mask);
    dependents_may_start();
    const long long rows = (long long) n * heads * d, total = rows * cells;
    const int pieces = (cells + ATTN_JOIN_CELLS - 1) / ATTN_JOIN_CELLS;
    for (long long u = blockIdx.x; u < rows * pieces; u += gridDim.x)
    {
        const long long row = u / pieces, b = row / ((long long) heads * d);
        const int i0 = (int) (u - row * pieces) * ATTN_JOIN_CELLS + threadIdx.x;
        const float* from = part + row * cells;
        T* to = static_cast<T*>(t.p) + b * t.sn + (row - b * heads * d) * t.sc;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        bool there[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            there[e] = i0 + 256 * e < cells && (!mask || mask[b * cells + i0 + 256 * e]);
#pragma unroll 2
        for (int s = 0; s < splits; ++s, from += total)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (there[e])
                    sum[e] += from[i0 + 256 * e];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i0 + 256 * e < cells)
            {
                const float v[1] = {sum[e]};
                store_elems<1>(to + i0 + 256 * e, v);
            }
    }
}

constexpr int ATTN_STATS_CELLS = 64, ATTN_STATS_WARPS = 8; // of a block: two cells a lane, an eighth of the channels a warp

// stats: lse in powers of two and delta = sum_c o d_o; a cell that takes no part has +infinity and 0, so that its
// weights are exp2(s - infinity) = 0.  2 x 4096 cells, 8 heads of 64 channels: 8 us, 14 with a condition at each load,
// 19 with a thread a cell.
template <class T>
__global__ void __launch_bounds__(32 * ATTN_STATS_WARPS) attn_stats_kernel(AttnProblem p)
{
    __shared__ float part[ATTN_STATS_WARPS][ATTN_STATS_CELLS];
    wait_for_previous_kernel(p.lse);
    dependents_may_start();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long heads = (long long) p.n * p.q_heads;
    const int chunks = (int) ((p.stats_pitch + ATTN_STATS_CELLS - 1) / ATTN_STATS_CELLS);
    for (long long at = blockIdx.x; at < heads * chunks; at += gridDim.x)
    {
        const long long nh = at / chunks, n = nh / p.q_heads, first = (nh - n * p.q_heads) * p.d;
        const int i0 = (int) (at - nh * chunks) * ATTN_STATS_CELLS;
        const int* index = p.q_side.index ? p.q_side.index + n * p.sq : nullptr;
        const int count = index ? p.q_side.count[n] : p.sq;
        const T* o = static_cast<const T*>(p.o.p) + n * p.o.sn + first * p.o.sc;
        const T* g = static_cast<const T*>(p.d_o.p) + n * p.d_o.sn + first * p.d_o.sc;
        bool there[2];
        int cell[2];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e)
        {
            const int r = i0 + lane + 32 * e;
            there[e] = r < count;
            cell[e] = !there[e] ? 0 : index ? index[r] : r;
        }
        // eight channels' loads go out without a condition (cell 0, the last channel) before the first is waited for
        for (int c0 = warp; c0 < p.d; c0 += 8 * ATTN_STATS_WARPS)
        {
            RawElems<T, 1> a[8][2], b[8][2];
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                const int c = min(c0 + ATTN_STATS_WARPS * k, p.d - 1);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                {
                    a[k][e].load(o + c * p.o.sc + cell[e]);
                    b[k][e].load(g + c * p.d_o.sc + cell[e]);
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c0 + ATTN_STATS_WARPS * k < p.d)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        sum[e] = fmaf(a[k][e].get(0), b[k][e].get(0), sum[e]);
        }
        part[warp][lane] = there[0] ? sum[0] : 0.f;
        part[warp][lane + 32] = there[1] ? sum[1] : 0.f;
        __syncthreads();
        const int i = i0 + (int) threadIdx.x;
        if (threadIdx.x < ATTN_STATS_CELLS && i < p.stats_pitch)
        {
            float delta = 0.f;
            for (int w = 0; w < ATTN_STATS_WARPS; ++w)
                delta += part[w][threadIdx.x];
            const int at_cell = i < count && index ? index[i] : i;
            const float lse = i < count ? p.lse[nh * p.sq + at_cell] : -INFINITY;
            const bool none = lse == -INFINITY;
            p.stats[nh * p.stats_pitch + i] = none ? INFINITY : lse * ATTN_LOG2E;
            p.stats[heads * p.stats_pitch + nh * p.stats_pitch + i] = none ? 0.f : delta;
        }
        __syncthreads();
    }
}

// Zeros, and lse of a cell that sees nothing.
template <class T>
__global__ void __launch_bounds__(256) attn_fill_kernel(AttnTensor t, int n, long long channels, int cells, float* lse,
                                                        long long lse_count)
{
    const long long total = n * channels * cells;
    const long long at0 = (long long) blockIdx.x * 256 + threadIdx.x, step = (long long) gridDim.x * 256;
    for (long long at = at0; at < total; at += step)
    {
        const long long row = at / cells, b = row / channels;
        const float v[1] = {0.f};
        store_elems<1>(static_cast<T*>(t.p) + b * t.sn + (row - b * channels) * t.sc + (at - row * cells), v);
    }
    if (lse)
        for (long long at = at0; at < lse_count; at += step)
            lse[at] = -INFINITY;
}

unsigned flat_blocks(long long total, int threads)
{
    return (unsigned) std::max<long long>(1, std::min<long long>((total + threads - 1) / threads, 16ll * num_sms()));
}

template <class F>
int32_t with_type(int32_t dtype, F f)
{
    return dtype == DCB_BF16 ? f(bf16()) : f(float());
}

int32_t attn_fill(int32_t dtype, const AttnTensor& t, int n, long long channels, int cells, float* lse,
                  long long lse_count, cudaStream_t s)
{
    return with_type(dtype, [&](auto e) -> int32_t {
        const long long total = std::max(n * channels * cells, lse ? lse_count : 0);
        if (total == 0)
            return DCB_OK;
        attn_fill_kernel<decltype(e)><<<flat_blocks(total, 256), 256, 0, s>>>(t, n, channels, cells, lse, lse_count);
        DCB_LAUNCH_CHECK();
        return DCB_OK;
    });
}

// Of a sample; 2^40 stands for all numbers from there on, whatever their product wraps to.
int64_t cells_of(const dcb_nd_desc& d)
{
    constexpr int64_t MANY = 1ll << 40;
    int64_t cells = 1;
    for (int i = 0; i < 3; ++i)
        cells = cells == 0 || d.dims[i] == 0 ? 0 : d.dims[i] >= MANY / cells ? MANY : cells * d.dims[i];
    return cells;
}

// What follows from the shapes alone.
int32_t attn_shapes(const dcb_attention_desc* ad, const dcb_nd_desc* qd, const dcb_nd_desc* kd, AttnProblem* p)
{
    DCB_REQUIRE(ad, "null descriptor");
    if (int32_t e = check_nd_desc(qd))
        return e;
    if (int32_t e = check_nd_desc(kd))
        return e;
    DCB_REQUIRE(known_dtype(ad->dtype), "dtype must be DCB_F32 or DCB_BF16");
    DCB_REQUIRE(ad->q_heads >= 1 && ad->kv_heads >= 1 && ad->q_heads % ad->kv_heads == 0,
                "q_heads must be a multiple of kv_heads");
    DCB_REQUIRE(qd->c >= 1 && qd->c % ad->q_heads == 0, "channels of q must be q_heads heads");
    const int64_t d = qd->c / ad->q_heads;
    DCB_REQUIRE(kd->c == d * ad->kv_heads, "channels of k must be kv_heads heads of q's size");
    DCB_REQUIRE(qd->n == kd->n, "q and k differ in samples");
    DCB_REQUIRE(ad->scale > 0.f && std::isfinite(ad->scale * ATTN_LOG2E),
                "scale must be positive, and finite times log2(e)");
    if (d > ATTN_MAX_HEAD)
    {
        set_last_error("unsupported: heads of more than 128 channels");
        return DCB_UNSUPPORTED;
    }
    if (cells_of(*qd) >= (1ll << 30) || cells_of(*kd) >= (1ll << 30) || qd->n >= (1ll << 24) || ad->q_heads >= (1 << 16))
    {
        set_last_error("unsupported: 2^30 cells of a sample, 2^24 samples or 2^16 heads");
        return DCB_UNSUPPORTED;
    }
    *p = AttnProblem();
    p->n = (int) qd->n;
    p->q_heads = ad->q_heads;
    p->kv_heads = ad->kv_heads;
    p->group = ad->q_heads / ad->kv_heads;
    p->d = (int) d;
    p->sq = (int) cells_of(*qd);
    p->sk = (int) cells_of(*kd);
    p->causal = ad->causal != 0;
    p->offset = p->sk - p->sq;
    p->scale = ad->scale * ATTN_LOG2E;
    return DCB_OK;
}

int32_t attn_tensor(const dcb_nd_desc* d, const dcb_nd_desc* like, const void* ptr, const char* name, AttnTensor* t)
{
    if (int32_t e = check_nd_desc(d))
        return e;
    if (!same_extents(*d, *like))
    {
        set_last_error(std::string("bad argument: extents of ") + name);
        return DCB_BAD_ARG;
    }
    if (run_level(*d) != 2)
    {
        set_last_error(std::string("unsupported: the cells of ") + name + " are not contiguous");
        return DCB_UNSUPPORTED;
    }
    if (cells_of(*d) > 0 && d->n > 0)
        DCB_REQUIRE(ptr, "null tensor");
    *t = AttnTensor{const_cast<void*>(ptr), d->sn, d->sc};
    return DCB_OK;
}

// The memory of an operand or a result, in bytes: n x c rows.
struct AttnRows
{
    const char* p;
    int64_t n, c, sn, sc, row;
    int64_t first() const { return std::min<int64_t>(0, (n - 1) * sn) + std::min<int64_t>(0, (c - 1) * sc); }
    int64_t last() const { return std::max<int64_t>(0, (n - 1) * sn) + std::max<int64_t>(0, (c - 1) * sc) + row; }
};

AttnRows attn_rows(const AttnTensor& t, int32_t dtype, const dcb_nd_desc& d)
{
    const int64_t es = elem_bytes(dtype);
    return AttnRows{static_cast<const char*>(t.p), d.n, d.c, t.sn * es, t.sc * es, cells_of(d) * es};
}

AttnRows attn_rows(const void* p, int64_t bytes)
{
    return AttnRows{static_cast<const char*>(p), 1, 1, 0, 0, bytes};
}

// Whether they share a byte.  Rows with the same strides (slices of one packed tensor) are compared one by one, others by
// their extent.
bool attn_overlap(AttnRows a, AttnRows b)
{
    for (const AttnRows* r : {&a, &b})
        if (!r->p || r->n == 0 || r->c == 0 || r->row == 0)
            return false;
    // how far b's first row lies behind a's: addresses may be anything
    const int64_t apart = (int64_t) (reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
    if (apart + b.first() >= a.last() || apart + b.last() <= a.first())
        return false;
    // a stride that nothing steps over is the other's
    if (a.n == 1)
        a.sn = b.n == 1 ? 0 : b.sn;
    if (b.n == 1)
        b.sn = a.sn;
    if (a.c == 1)
        a.sc = b.c == 1 ? 0 : b.sc;
    if (b.c == 1)
        b.sc = a.sc;
    if (a.sc > a.sn) // the longer steps first
        for (AttnRows* r : {&a, &b})
            std::swap(r->n, r->c), std::swap(r->sn, r->sc);
    if (a.sn != b.sn || a.sc != b.sc || a.sn < 0 || a.sc < 0)
        return true;
    // rows i, j of a and i + k, j + l of b share a byte if apart + k sn + l sc lies in (-b.row, a.row)
    const auto near = [](int64_t at, int64_t step, int64_t lo, int64_t hi, int64_t below, int64_t above, auto f) {
        // every k in [lo, hi] with at + k step in (below, above)
        if (step > 0)
        {
            const auto floor_div = [](int64_t x, int64_t d) { return x >= 0 ? x / d : -((-x + d - 1) / d); };
            lo = std::max(lo, floor_div(below - at, step) + 1);
            hi = std::min(hi, -floor_div(at - above, step) - 1);
        }
        else if (at <= below || at >= above)
            return false;
        else
            hi = std::min(hi, lo);
        for (int64_t k = lo; k <= hi; ++k)
            if (f(at + k * step))
                return true;
        return false;
    };
    const int64_t reach = a.sc * std::max(a.c, b.c);
    return near(apart, a.sn, 1 - a.n, b.n - 1, -b.row - reach, a.row + reach, [&](int64_t at) {
        return near(at, a.sc, 1 - a.c, b.c - 1, -b.row, a.row, [](int64_t) { return true; });
    });
}

// No result shares memory with an operand or another result.
int32_t attn_places(std::initializer_list<AttnRows> results, std::initializer_list<AttnRows> operands)
{
    for (auto r = results.begin(); r != results.end(); ++r)
    {
        for (const AttnRows& x : operands)
            DCB_REQUIRE(!attn_overlap(*r, x), "a result in an operand's place");
        for (auto other = r + 1; other != results.end(); ++other)
            DCB_REQUIRE(!attn_overlap(*r, *other), "two results in one place");
    }
    return DCB_OK;
}

// The workspace, piece by piece; a null base only counts.
struct Carve
{
    char* base;
    int64_t used = 0;
    float* floats(long long count)
    {
        float* p = base ? reinterpret_cast<float*>(base + used) : nullptr;
        used += (count * 4 + 255) / 256 * 256;
        return p;
    }
};

int64_t attn_carve(AttnProblem* p, int32_t dtype, bool backward, void* workspace)
{
    Carve w{static_cast<char*>(workspace)};
    const bool tc = dtype == DCB_BF16;
    const bool thin = backward ? attn_thin_backward(*p, dtype) : attn_thin(*p, dtype);
    if (thin && backward)
        attn_thin_bwd_splits(p);
    else if (thin)
        attn_thin_splits(p, dtype);
    else
        (tc ? attn_tc_splits : attn_simt_splits)(p, backward);
    const long long qh = (long long) p->n * p->q_heads, kh = (long long) p->n * p->kv_heads;
    p->stats_pitch = tc ? (long long) attn_tiles(p->sq, 128) * 128 : p->sq;
    const auto side = [&](int cells, bool masked) {
        AttnSide t;
        t.index = reinterpret_cast<int*>(w.floats((long long) p->n * cells));
        t.before = reinterpret_cast<int*>(w.floats((long long) p->n * (cells + 1)));
        t.count = reinterpret_cast<int*>(w.floats(p->n));
        return masked ? t : AttnSide{};
    };
    p->q_side = side(p->sq, p->q_mask != nullptr);
    p->kv_side = side(p->sk, p->kv_mask != nullptr);
    if (tc && !thin)
    {
        const auto copy = [&](long long heads, int cells) {
            return reinterpret_cast<bf16*>(w.floats(heads * p->d * ((cells + 7) / 8) * 4));
        };
        p->copy_q = copy(qh, p->sq);
        p->copy_k = copy(kh, p->sk);
        p->copy_v = copy(kh, p->sk);
        p->copy_do = backward ? copy(qh, p->sq) : nullptr;
    }
    if (!backward)
    {
        if (p->kv_splits > 1)
        {
            p->part_o = w.floats(p->kv_splits * qh * p->d * p->sq);
            p->part_ml = w.floats(p->kv_splits * 2 * qh * p->sq);
        }
        return w.used;
    }
    p->stats = w.floats(2 * qh * p->stats_pitch);
    if (p->kv_splits > 1)
        p->part_dq = w.floats(p->kv_splits * qh * p->d * p->sq);
    if (p->q_splits > 1)
    {
        p->part_dk = w.floats(p->q_splits * kh * p->d * p->sk);
        p->part_dv = w.floats(p->q_splits * kh * p->d * p->sk);
    }
    return w.used;
}

int32_t attn_workspace(AttnProblem* p, int32_t dtype, bool backward, void* workspace, int64_t bytes)
{
    const int64_t need = attn_carve(p, dtype, backward, nullptr);
    if (need > 0)
    {
        DCB_REQUIRE(workspace && bytes >= need, "workspace too small");
        DCB_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 256 == 0, "workspace must be 256-byte aligned");
        attn_carve(p, dtype, backward, workspace);
    }
    return DCB_OK;
}

int32_t attn_join_grad(int32_t dtype, const float* part, int splits, const AttnTensor& t, int n, int heads, int d,
                       int cells, const uint8_t* mask, cudaStream_t s)
{
    return with_type(dtype, [&](auto e) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(attn_join_grad_kernel<decltype(e)>,
                                       dim3((unsigned) std::min<long long>((long long) n * heads * d
                                                                               * ((cells + ATTN_JOIN_CELLS - 1) / ATTN_JOIN_CELLS),
                                                                           32ll * num_sms())),
                                       256, 0, s, part,
                                       splits, t, n, heads, d, cells, mask));
        return DCB_OK;
    });
}

// What the masks leave of both sides.
int32_t attn_index(const AttnProblem& p, cudaStream_t s)
{
    if (!p.q_mask && !p.kv_mask)
        return DCB_OK;
    const int steps = attn_tiles(std::max(p.q_mask ? p.sq : 0, p.kv_mask ? p.sk : 0), ATTN_INDEX_THREADS * ATTN_INDEX_CELLS);
    const dim3 grid(p.n, 2, std::max(1, std::min(steps, ATTN_INDEX_PARTS)));
    DCB_CUDA_TRY(launch_overlapped(attn_index_kernel, grid, ATTN_INDEX_THREADS, 0, s, p));
    return DCB_OK;
}

// The results' cells that the masks take out, of those that no join writes.
int32_t attn_zeros(const AttnProblem& p, int32_t dtype, bool backward, cudaStream_t s)
{
    AttnZeroJobs a = {};
    int jobs = 0;
    long long units = 0;
    const auto add = [&](const AttnTensor& t, int heads, int cells, const uint8_t* mask, float* lse) {
        if (!mask)
            return;
        a.job[jobs++] = AttnZeros{t, mask, (long long) heads * p.d, cells, lse, lse ? heads : 0};
        units = std::max(units, (long long) p.n * (heads * (p.d + 1ll) / ATTN_ZERO_ROWS + 1) * ((cells + 255) / 256));
    };
    if (!backward && p.kv_splits == 1)
        add(p.o, p.q_heads, p.sq, p.q_mask, p.lse);
    if (backward && p.kv_splits == 1)
        add(p.dq, p.q_heads, p.sq, p.q_mask, nullptr);
    if (backward && p.q_splits == 1)
    {
        add(p.dk, p.kv_heads, p.sk, p.kv_mask, nullptr);
        add(p.dv, p.kv_heads, p.sk, p.kv_mask, nullptr);
    }
    if (jobs == 0)
        return DCB_OK;
    a.n = p.n;
    return with_type(dtype, [&](auto e) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(attn_zero_kernel<decltype(e)>,
                                       dim3((unsigned) std::min<long long>(units, 16ll * num_sms()), jobs), 256, 0, s,
                                       a));
        return DCB_OK;
    });
}

} // namespace
} // namespace dcb

using namespace dcb;

extern "C" {

int64_t dcb_attention_workspace_bytes(const dcb_attention_desc* ad, const dcb_nd_desc* qd, const dcb_nd_desc* kd,
                                      int32_t backward)
{
    AttnProblem p;
    if (attn_shapes(ad, qd, kd, &p))
        return -1;
    const int64_t plain = attn_carve(&p, ad->dtype, backward != 0, nullptr);
    static const uint8_t any = 0;
    p.q_mask = p.kv_mask = &any; // only asked for: masked walks may be cut in other parts
    return std::max(plain, attn_carve(&p, ad->dtype, backward != 0, nullptr));
}

int32_t dcb_attention_fwd(const dcb_attention_desc* ad, const dcb_nd_desc* qd, const void* q, const dcb_nd_desc* kd,
                          const void* k, const dcb_nd_desc* vd, const void* v, const void* q_mask, const void* kv_mask,
                          const dcb_nd_desc* od, void* o, void* lse, void* workspace, int64_t workspace_bytes,
                          void* stream)
{
    AttnProblem p;
    if (int32_t e = attn_shapes(ad, qd, kd, &p))
        return e;
    if (int32_t e = attn_tensor(qd, qd, q, "q", &p.q))
        return e;
    if (int32_t e = attn_tensor(kd, kd, k, "k", &p.k))
        return e;
    if (int32_t e = attn_tensor(vd, kd, v, "v", &p.v))
        return e;
    if (int32_t e = attn_tensor(od, qd, o, "o", &p.o))
        return e;
    if (p.n == 0 || p.sq == 0)
        return DCB_OK;
    DCB_REQUIRE(lse, "null lse");
    const int64_t cells_q = (int64_t) p.n * p.sq, cells_k = (int64_t) p.n * p.sk;
    if (int32_t e = attn_places({attn_rows(p.o, ad->dtype, *qd), attn_rows(lse, 4 * p.q_heads * cells_q)},
                                {attn_rows(p.q, ad->dtype, *qd), attn_rows(p.k, ad->dtype, *kd),
                                 attn_rows(p.v, ad->dtype, *kd), attn_rows(q_mask, cells_q), attn_rows(kv_mask, cells_k)}))
        return e;
    cudaStream_t s = as_stream(stream);
    p.lse = static_cast<float*>(lse);
    p.q_mask = static_cast<const uint8_t*>(q_mask);
    p.kv_mask = static_cast<const uint8_t*>(kv_mask);
    if (p.sk == 0)
        return attn_fill(ad->dtype, p.o, p.n, (long long) p.q_heads * p.d, p.sq, p.lse,
                         (long long) p.n * p.q_heads * p.sq, s);
    if (int32_t e = attn_workspace(&p, ad->dtype, false, workspace, workspace_bytes))
        return e;
    if (int32_t e = attn_index(p, s))
        return e;
    if (int32_t e = attn_zeros(p, ad->dtype, false, s))
        return e;
    const int32_t e = attn_thin(p, ad->dtype)   ? attn_thin_fwd(p, ad->dtype, s)
                      : ad->dtype == DCB_BF16 ? attn_tc_fwd(p, s)
                                              : attn_simt_fwd(p, s);
    if (e)
        return e;
    if (p.kv_splits == 1)
        return DCB_OK;
    return with_type(ad->dtype, [&](auto t) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(attn_join_fwd_kernel<decltype(t)>,
                                       dim3(flat_blocks((long long) p.n * p.q_heads * p.d * p.sq, 256)), 256, 0, s, p));
        return DCB_OK;
    });
}

int32_t dcb_attention_bwd(const dcb_attention_desc* ad, const dcb_nd_desc* qd, const void* q, const dcb_nd_desc* kd,
                          const void* k, const dcb_nd_desc* vd, const void* v, const void* q_mask, const void* kv_mask,
                          const dcb_nd_desc* od, const void* o, const void* lse, const dcb_nd_desc* dod,
                          const void* d_o, const dcb_nd_desc* dqd, void* dq, const dcb_nd_desc* dkd, void* dk,
                          const dcb_nd_desc* dvd, void* dv, void* workspace, int64_t workspace_bytes, void* stream)
{
    AttnProblem p;
    if (int32_t e = attn_shapes(ad, qd, kd, &p))
        return e;
    const struct
    {
        const dcb_nd_desc *d, *like;
        const void* ptr;
        const char* name;
        AttnTensor* to;
    } tensors[] = {{qd, qd, q, "q", &p.q},    {kd, kd, k, "k", &p.k},      {vd, kd, v, "v", &p.v},
                   {od, qd, o, "o", &p.o},    {dod, qd, d_o, "d_o", &p.d_o}, {dqd, qd, dq, "dq", &p.dq},
                   {dkd, kd, dk, "dk", &p.dk}, {dvd, kd, dv, "dv", &p.dv}};
    for (const auto& t : tensors)
        if (int32_t e = attn_tensor(t.d, t.like, t.ptr, t.name, t.to))
            return e;
    if (p.n == 0)
        return DCB_OK;
    const int64_t cells_q = (int64_t) p.n * p.sq, cells_k = (int64_t) p.n * p.sk;
    if (int32_t e = attn_places({attn_rows(p.dq, ad->dtype, *qd), attn_rows(p.dk, ad->dtype, *kd),
                                 attn_rows(p.dv, ad->dtype, *kd)},
                                {attn_rows(p.q, ad->dtype, *qd), attn_rows(p.k, ad->dtype, *kd),
                                 attn_rows(p.v, ad->dtype, *kd), attn_rows(p.o, ad->dtype, *qd),
                                 attn_rows(p.d_o, ad->dtype, *qd), attn_rows(lse, 4 * p.q_heads * cells_q),
                                 attn_rows(q_mask, cells_q), attn_rows(kv_mask, cells_k)}))
        return e;
    cudaStream_t s = as_stream(stream);
    if (p.sq == 0 || p.sk == 0) // one side is empty: the other's gradients are zero
    {
        if (int32_t e = attn_fill(ad->dtype, p.dq, p.n, (long long) p.q_heads * p.d, p.sq, nullptr, 0, s))
            return e;
        if (int32_t e = attn_fill(ad->dtype, p.dk, p.n, (long long) p.kv_heads * p.d, p.sk, nullptr, 0, s))
            return e;
        return attn_fill(ad->dtype, p.dv, p.n, (long long) p.kv_heads * p.d, p.sk, nullptr, 0, s);
    }
    DCB_REQUIRE(lse, "null lse");
    p.lse = static_cast<float*>(const_cast<void*>(lse));
    p.q_mask = static_cast<const uint8_t*>(q_mask);
    p.kv_mask = static_cast<const uint8_t*>(kv_mask);
    if (int32_t e = attn_workspace(&p, ad->dtype, true, workspace, workspace_bytes))
        return e;
    if (int32_t err = attn_index(p, s))
        return err;
    if (int32_t err = attn_zeros(p, ad->dtype, true, s))
        return err;
    const int32_t e = with_type(ad->dtype, [&](auto t) -> int32_t {
        DCB_CUDA_TRY(launch_overlapped(attn_stats_kernel<decltype(t)>,
                                       dim3((unsigned) std::min<long long>(
                                           (long long) p.n * p.q_heads
                                               * ((p.stats_pitch + ATTN_STATS_CELLS - 1) / ATTN_STATS_CELLS),
                                           8ll * num_sms())),
                                       32 * ATTN_STATS_WARPS, 0, s, p));
        return DCB_OK;
    });
    if (e)
        return e;
    const int32_t err = attn_thin_backward(p, ad->dtype) ? attn_thin_bwd(p, s)
                        : ad->dtype == DCB_BF16   ? attn_tc_bwd(p, s)
                                                  : attn_simt_bwd(p, s);
    if (err)
        return err;
    if (p.q_splits > 1)
    {
        if (int32_t err = attn_join_grad(ad->dtype, p.part_dk, p.q_splits, p.dk, p.n, p.kv_heads, p.d, p.sk, p.kv_mask, s))
            return err;
        if (int32_t err = attn_join_grad(ad->dtype, p.part_dv, p.q_splits, p.dv, p.n, p.kv_heads, p.d, p.sk, p.kv_mask, s))
            return err;
    }
    if (p.kv_splits > 1)
        return attn_join_grad(ad->dtype, p.part_dq, p.kv_splits, p.dq, p.n, p.q_heads, p.d, p.sq, p.q_mask, s);
    return DCB_OK;
}

int32_t dcb_attention_status(void* stream)
{
    DCB_CUDA_TRY(cudaStreamSynchronize(as_stream(stream)));
    bool gave_up = false;
    if (int32_t e = attn_tc_status(&gave_up))
        return e;
    if (!gave_up)
        return DCB_OK;
    set_last_error("a tensor-core attention kernel gave up on a pipeline wait");
    return DCB_CUDA_ERROR;
}

} // extern "C"
