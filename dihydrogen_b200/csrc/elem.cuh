// Element types of the kernels that take more than fp32: loads of V neighbours as floats,
// stores rounded to nearest even.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

#include <algorithm>

namespace dcb
{

typedef __nv_bfloat16 bf16;

inline int elem_bytes(int32_t dtype)
{
    return dtype == DCB_BF16 ? 2 : 4;
}

inline bool known_dtype(int32_t dtype)
{
    return dtype == DCB_F32 || dtype == DCB_BF16;
}

// Largest of `most` (8 or 4), 4, 2, 1 elements that every run start of a tensor honours as accesses of 16 bytes or less.
inline int run_vec_of(const RunGeom& g, const RunStrides& s, const void* p, int bytes, int most = 4)
{
    auto ok = [&](long long v) {
        const long long aligned = std::min<long long>(v, 16 / bytes); // elements
        return g.len % v == 0 && s.sn % aligned == 0 && s.sc % aligned == 0 && s.s_inner % aligned == 0
               && s.s_outer % aligned == 0 && reinterpret_cast<uintptr_t>(p) % (bytes * aligned) == 0;
    };
    return most == 8 && ok(8) ? 8 : ok(4) ? 4 : (ok(2) ? 2 : 1);
}

// A row's stride that nothing ever steps over says nothing about alignment.
inline void drop_unused_strides(const RunGeom& g, RunStrides* s)
{
    if (g.n <= 1)
        s->sn = 0;
    if (g.c <= 1)
        s->sc = 0;
    if (g.rows_inner <= 1)
        s->s_inner = 0;
    if (g.rows <= g.rows_inner)
        s->s_outer = 0;
}

template <int V>
__device__ __forceinline__ void load_elems(const float* p, float (&v)[V])
{
    if constexpr (V == 4)
    {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    }
    else if constexpr (V == 2)
    {
        const float2 t = *reinterpret_cast<const float2*>(p);
        v[0] = t.x, v[1] = t.y;
    }
    else
        v[0] = *p;
}

template <int V>
__device__ __forceinline__ void load_elems(const bf16* p, float (&v)[V])
{
    if constexpr (V == 4)
    {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(t.x << 16), v[1] = __uint_as_float(t.x & 0xffff0000u);
        v[2] = __uint_as_float(t.y << 16), v[3] = __uint_as_float(t.y & 0xffff0000u);
    }
    else if constexpr (V == 2)
    {
        const uint32_t t = *reinterpret_cast<const uint32_t*>(p);
        v[0] = __uint_as_float(t << 16), v[1] = __uint_as_float(t & 0xffff0000u);
    }
    else
        v[0] = __bfloat162float(*p);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi)
{
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

template <>
__device__ __forceinline__ void load_elems<8>(const float* p, float (&v)[8])
{
    const float4 t = *reinterpret_cast<const float4*>(p), u = *reinterpret_cast<const float4*>(p + 4);
    v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w, v[4] = u.x, v[5] = u.y, v[6] = u.z, v[7] = u.w;
}

// V neighbours as they are stored.  Loads that are taken ahead keep these and are converted where they are used: a
// conversion right behind a load waits for it.
template <class T, int V>
struct RawElems;

template <int V>
struct RawElems<float, V>
{
    float v[V];
    __device__ __forceinline__ void load(const float* p) { load_elems<V>(p, v); }
    __device__ __forceinline__ float get(int e) const { return v[e]; }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int e = 0; e < V; ++e)
            v[e] = 0.f;
    }
};

template <int V>
struct RawElems<bf16, V>
{
    static constexpr int WORDS = (V + 1) / 2;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const bf16* p)
    {
        if constexpr (V == 8)
        {
            const uint4 t = *reinterpret_cast<const uint4*>(p);
            w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
        }
        else if constexpr (V == 4)
        {
            const uint2 t = *reinterpret_cast<const uint2*>(p);
            w[0] = t.x, w[1] = t.y;
        }
        else if constexpr (V == 2)
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        else
            w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
    __device__ __forceinline__ float get(int e) const
    {
        return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    }
    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < WORDS; ++i)
            w[i] = 0;
    }
};

template <int V>
__device__ __forceinline__ void store_elems(float* p, const float (&v)[V])
{
    if constexpr (V == 8)
    {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
    else if constexpr (V == 4)
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (V == 2)
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else
        *p = v[0];
}

template <int V>
__device__ __forceinline__ void store_elems(bf16* p, const float (&v)[V])
{
    if constexpr (V == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]),
                                                  pack_bf16(v[6], v[7]));
    else if constexpr (V == 4)
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    else if constexpr (V == 2)
        *reinterpret_cast<uint32_t*>(p) = pack_bf16(v[0], v[1]);
    else
        *p = __float2bfloat16_rn(v[0]);
}

// V elements 32 apart, of which the first `have` are there: a lane's share of 32 V neighbours where a run starts off the
// alignment of wider accesses.  They share an address but for a constant.
template <class T, int V>
struct SplitElems
{
    RawElems<T, 1> r[V];
    template <bool FULL>
    __device__ __forceinline__ void load(const T* p, int have)
    {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (FULL || e < have)
                r[e].load(p + 32 * e);
            else
                r[e].clear();
    }
    __device__ __forceinline__ float get(int e) const { return r[e].get(0); }
};

template <int V, bool FULL, class T>
__device__ __forceinline__ void store_split(T* p, const float (&v)[V], int have)
{
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (FULL || e < have)
        {
            const float t[1] = {v[e]};
            store_elems<1>(p + 32 * e, t);
        }
}

// Units of V neighbouring cells of all samples, numbered through: which cells a unit is.
struct CellUnits
{
    long long total;   // units in all
    long long cells;   // cells of a sample
    long long len;     // cells of a run
    FastDiv per_run, rows, rows_inner;
    int narrow;        // all numbers have 31 bits
};

// `per_run` units a run.
inline CellUnits cell_units_of(const RunGeom& g, long long per_run)
{
    CellUnits u;
    u.total = g.n * g.rows * per_run;
    u.cells = g.rows * g.len;
    u.len = g.len;
    u.narrow = u.total < (1ll << 31);
    const auto safe = [](long long d) { return FastDiv::of((uint32_t) (d > 0 && d < (1ll << 31) ? d : 1)); };
    u.per_run = safe(per_run);
    u.rows = safe(g.rows);
    u.rows_inner = safe(g.rows_inner);
    return u;
}

struct CellAt
{
    long long n;
    uint32_t outer, inner; // row of the sample, by the two steps
    long long pos;         // first cell within the run
    long long cell;        // first cell of the sample, dense
};

template <int V>
__device__ __forceinline__ CellAt cell_at(const CellUnits& g, long long per_run, long long rows, long long rows_inner,
                                          long long unit)
{
    CellAt a;
    long long row, in_run;
    if (g.narrow)
    {
        const uint32_t u = (uint32_t) unit;
        const uint32_t r = g.per_run.div(u);
        in_run = u - r * g.per_run.d;
        const uint32_t n = g.rows.div(r);
        row = r - n * g.rows.d;
        a.n = n;
        a.outer = g.rows_inner.div((uint32_t) row);
        a.inner = (uint32_t) row - a.outer * g.rows_inner.d;
    }
    else
    {
        const long long r = unit / per_run;
        in_run = unit - r * per_run;
        a.n = r / rows;
        row = r - a.n * rows;
        a.outer = (uint32_t) (row / rows_inner);
        a.inner = (uint32_t) (row - a.outer * rows_inner);
    }
    a.pos = in_run * V;
    a.cell = row * g.len + a.pos;
    return a;
}

__device__ __forceinline__ long long offset_of(const CellAt& a, const RunStrides& s)
{
    return a.n * s.sn + a.outer * s.s_outer + a.inner * s.s_inner + a.pos;
}

// Sums over a warp's lanes of K values a lane, by halves: lane l ends with the sum of value l mod K
// in v[0].  K - 1 + log2(32 / K) exchanges instead of 5 K.
template <int K>
__device__ __forceinline__ float lane_sums(float (&v)[K], int lane)
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

} // namespace dcb
