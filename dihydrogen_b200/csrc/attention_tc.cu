// Attention on the tensor cores, host side: what has to be copied first, tensor maps, the status word.
#include "attention_tc.cuh"
#include "conv_tc_encode.cuh"

#include <cmath>

namespace dcb
{
namespace
{

constexpr int AT_JOBS = 4;
constexpr int AT_ROWS = 8; // rows of a tensor that a warp copies with the same indices
// A copy with rows of whole 16 bytes, of the cells that a mask leaves; zeros behind the last.
struct AtJob
{
    const bf16* from;
    bf16* to;
    long long sn, sc;
    AttnSide side;
    int channels, cells; // rows of a sample
    int chunks;          // of 256 cells a row: a warp each
};

struct AtPrepare
{
    AtJob job[AT_JOBS];
    int jobs;
    int n;
};

__global__ void __launch_bounds__(256) attn_prepare_kernel(const __grid_constant__ AtPrepare a)
{
    const AtJob& c = a.job[blockIdx.y];
    const bf16* source = c.from;
    wait_for_previous_kernel(source);
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const int groups = (c.channels + AT_ROWS - 1) / AT_ROWS;
    const long long total = (long long) a.n * groups * c.chunks;
    const int pitch = (c.cells + 7) / 8 * 8;
    for (long long u = (long long) blockIdx.x * 8 + (threadIdx.x >> 5); u < total; u += (long long) gridDim.x * 8)
    {
        const long long m = u / c.chunks, n = m / groups;
        const int row0 = (int) (m - n * groups) * AT_ROWS, row1 = min(row0 + AT_ROWS, c.channels);
        const int i0 = (int) (u - m * c.chunks) * 256 + lane;
        const int count = c.side.index ? c.side.count[n] : c.cells;
        int cell[8]; // negative: nothing
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            const int i = i0 + 32 * e;
            cell[e] = i >= count ? -1 : c.side.index ? c.side.index[n * c.cells + i] : i;
        }
        for (int row = row0; row < row1; ++row)
        {
            const uint16_t* from = reinterpret_cast<const uint16_t*>(source) + n * c.sn + row * c.sc;
            uint16_t* to = reinterpret_cast<uint16_t*>(c.to) + (n * c.channels + row) * (long long) pitch + i0;
            uint16_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = cell[e] >= 0 ? from[cell[e]] : (uint16_t) 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i0 + 32 * e < pitch)
                    to[32 * e] = v[e];
        }
    }
}

struct AtHost
{
    AtPrepare prepare = {};
    AtMaps maps;
};

// The tensor as bulk copies see it, copied first where they cannot or where a mask picks cells.
int32_t at_operand(const AttnProblem& p, const AttnTensor& t, int heads, int cells, const AttnSide& side, bf16* copy,
                   int box_channels, AtHost* h, CUtensorMap* map)
{
    const void* at = t.p;
    long long sc = t.sc, sn = t.sn;
    const bool fits = reinterpret_cast<uintptr_t>(at) % 16 == 0 && sc % 8 == 0 && (p.n == 1 || sn % 8 == 0) && sc > 0
                      && (p.n == 1 || sn > 0);
    if (!fits || side.index)
    {
        const int channels = heads * p.d;
        h->prepare.job[h->prepare.jobs++]
            = AtJob{static_cast<const bf16*>(at), copy, sn, sc, side, channels, cells, (cells + 255) / 256};
        at = copy;
        sc = (cells + 7) / 8 * 8;
        sn = sc * channels;
    }
    const cuuint64_t dims[4] = {(cuuint64_t) cells, (cuuint64_t) p.d, (cuuint64_t) heads, (cuuint64_t) p.n};
    // a dimension of extent 1 may carry any stride; give it a valid one
    const cuuint64_t strides[3] = {(cuuint64_t) sc * 2, (cuuint64_t) (sc * p.d) * 2,
                                   (cuuint64_t) (p.n > 1 ? sn : sc * p.d * heads) * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t) box_channels, 1, 1}, one[4] = {1, 1, 1, 1};
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn
        || fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(at), dims, strides, box, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
               != CUDA_SUCCESS)
    {
        set_last_error("unsupported: attention tensor map");
        return DCB_UNSUPPORTED;
    }
    return DCB_OK;
}

int32_t at_prepare(const AttnProblem& p, AtHost* h, cudaStream_t stream)
{
    AtPrepare& a = h->prepare;
    if (a.jobs == 0)
        return DCB_OK;
    a.n = p.n;
    long long warps = 0;
    for (int i = 0; i < a.jobs; ++i)
        warps = std::max(warps, (long long) a.n * ((a.job[i].channels + AT_ROWS - 1) / AT_ROWS) * a.job[i].chunks);
    const unsigned blocks = (unsigned) std::min<long long>((warps + 7) / 8, 16ll * num_sms());
    DCB_CUDA_TRY(launch_overlapped(attn_prepare_kernel, dim3(blocks, a.jobs), 256, 0, stream, a));
    return DCB_OK;
}

} // namespace

int32_t attn_tc_status(bool* gave_up)
{
    *gave_up = false;
    if (int32_t e = attn_tc_fwd_status(gave_up))
        return e;
    return attn_tc_bwd_status(gave_up);
}

// 100 queries, 2 x 8 heads of 64: 32768 keys 46.5 us so and 50.6 with two tiles of queries, 4096 18.4 and 20.6, 2048 17.7
// and 17.7.  Heads of 128 have the room for one block an SM either way: 4096 keys 30.3 and 24.7.
bool attn_tc_apart(const AttnProblem& p)
{
    return p.sq <= AT_TILE && p.d <= 64 && attn_tiles(p.sk, AT_TILE) >= 32;
}

namespace
{

// In how many parts every walk is cut, for `work` walks of `steps` tiles of 128 cells on `slots` blocks at a time: what
// the longest of the slots' queues takes, with `step_us` a tile, and what the parts' sums of `part_bytes` a part cost.
// Causal walks are half as long on average and start with the longest, so that the queues are even but for one walk's
// length (12288 cells, 2 key heads of 128 channels: dk, dv in one part 617 us, in three 450).  Masks are taken to
// leave half of either side.
int at_best_splits(long long work, long long steps, long long slots, bool causal, bool masked, double step_us,
                   double part_bytes)
{
    const double left = masked ? 0.5 : 1.;
    int best = 1;
    double least = 0.;
    for (int s = 1; s <= 64 && (s == 1 || steps >= 2 * s); ++s)
    {
        const double length = std::ceil(left * steps / s);
        const double blocks = std::ceil(left * work * s / slots); // of a queue; each starts and ends for about 4 us
        const double queue = causal ? std::max(length, 0.5 * left * left * work * steps / slots) + 0.2 * length
                                    : blocks * length;
        const double us = queue * step_us + 4. * blocks + (s > 1 ? 4. + 2. * s * part_bytes / 4e6 : 0.);
        if (s == 1 || us < 0.97 * least)
            best = s, least = us;
    }
    return best;
}

} // namespace

void attn_tc_splits(AttnProblem* p, bool backward)
{
    const bool small = p->d <= 64, masked = p->q_mask || p->kv_mask;
    const long long slots = (small ? 2 : 1) * num_sms(); // blocks at a time
    const long long q_tiles = attn_tiles(p->sq, AT_TILE), k_tiles = attn_tiles(p->sk, AT_TILE);
    const long long qh = (long long) p->n * p->q_heads, kh = (long long) p->n * p->kv_heads;
    const double q_bytes = 4. * qh * p->d * p->sq, kv_bytes = 8. * kh * p->d * p->sk;
    p->q_splits = 1;
    if (backward)
    {
        p->kv_splits = at_best_splits(qh * q_tiles, k_tiles, slots, p->causal, masked, small ? 2.1 : 1., q_bytes);
        p->q_splits = at_best_splits(kh * k_tiles, q_tiles * p->group, slots, p->causal, masked, small ? 2.8 : 1.4,
                                     kv_bytes);
    }
    else if (attn_tc_apart(*p))
        p->kv_splits = 2 * at_best_splits(qh, k_tiles / 2, num_sms(), false, masked, 1.2, 2. * q_bytes);
    else
        p->kv_splits = at_best_splits(qh * ((q_tiles + 1) / 2), k_tiles, slots, p->causal, masked, small ? 3.4 : 2.1,
                                      q_bytes);
}

int32_t attn_tc_fwd(const AttnProblem& p, cudaStream_t stream)
{
    AtHost h;
    const int box = p.d <= 64 ? 64 : 128;
    if (int32_t e = at_operand(p, p.q, p.q_heads, p.sq, p.q_side, p.copy_q, box, &h, &h.maps.q))
        return e;
    if (int32_t e = at_operand(p, p.k, p.kv_heads, p.sk, p.kv_side, p.copy_k, box, &h, &h.maps.k))
        return e;
    if (int32_t e = at_operand(p, p.v, p.kv_heads, p.sk, p.kv_side, p.copy_v, box, &h, &h.maps.v))
        return e;
    h.maps.d_o = h.maps.q;
    if (int32_t e = at_prepare(p, &h, stream))
        return e;
    return attn_tc_fwd_launch(p, h.maps, stream);
}

int32_t attn_tc_bwd(const AttnProblem& p, cudaStream_t stream)
{
    AtHost h;
    const int box = p.d <= 64 ? 64 : 128;
    if (int32_t e = at_operand(p, p.q, p.q_heads, p.sq, p.q_side, p.copy_q, box, &h, &h.maps.q))
        return e;
    if (int32_t e = at_operand(p, p.k, p.kv_heads, p.sk, p.kv_side, p.copy_k, box, &h, &h.maps.k))
        return e;
    if (int32_t e = at_operand(p, p.v, p.kv_heads, p.sk, p.kv_side, p.copy_v, box, &h, &h.maps.v))
        return e;
    if (int32_t e = at_operand(p, p.d_o, p.q_heads, p.sq, p.q_side, p.copy_do, box, &h, &h.maps.d_o))
        return e;
    if (int32_t e = at_prepare(p, &h, stream))
        return e;
    return attn_tc_bwd_launch(p, h.maps, stream);
}

} // namespace dcb
