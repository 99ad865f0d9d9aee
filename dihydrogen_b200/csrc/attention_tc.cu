// Attention on the tensor cores, host side: what has to be copied first, tensor maps, the status word.
#include "attention_tc.cuh"
#include "conv_tc_encode.cuh"

namespace dcb
{
namespace
{

__device__ int at_status_word; // a kernel gave up on a wait

constexpr int AT_JOBS = 4;

// Copies with rows of whole 16 bytes; cells that a mask takes out, and those behind the last, as zeros.
struct AtCopy
{
    const bf16* from;
    bf16* to;
    long long sn, sc;
    const uint8_t* mask;
    int channels, cells;
    long long units; // of 8 cells, all samples
};

struct AtPrepare
{
    AtCopy job[AT_JOBS];
    int jobs;
    const uint8_t* mask; // to bits
    uint32_t* bits;
    int cells;
    long long words, words_total;
};

__global__ void __launch_bounds__(256) attn_prepare_kernel(const __grid_constant__ AtPrepare a)
{
    const uint8_t* mask = a.mask;
    wait_for_previous_kernel(mask);
    dependents_may_start();
    const long long step = (long long) gridDim.x * 256, first = (long long) blockIdx.x * 256 + threadIdx.x;
    if (blockIdx.y == (unsigned) a.jobs)
    {
        for (long long w = first; w < a.words_total; w += step)
        {
            const long long n = w / a.words;
            const long long j0 = (w - n * a.words) * 32;
            uint32_t bits = 0;
            for (int e = 0; e < 32; ++e)
                if (j0 + e < a.cells && mask[n * a.cells + j0 + e])
                    bits |= 1u << e;
            a.bits[w] = bits;
        }
        return;
    }
    const AtCopy& c = a.job[blockIdx.y];
    const int per_row = (c.cells + 7) / 8;
    for (long long u = first; u < c.units; u += step)
    {
        const long long row = u / per_row, n = row / c.channels;
        const int i0 = (int) (u - row * per_row) * 8;
        const bf16* from = c.from + n * c.sn + (row - n * c.channels) * c.sc + i0;
        uint32_t v[4];
#pragma unroll
        for (int e = 0; e < 8; ++e)
        {
            const bool there = i0 + e < c.cells && (!c.mask || c.mask[n * c.cells + i0 + e]);
            const uint32_t x = there ? reinterpret_cast<const uint16_t*>(from)[e] : 0u;
            v[e / 2] = e & 1 ? v[e / 2] | x << 16 : x;
        }
        reinterpret_cast<uint4*>(c.to)[u] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

struct AtHost
{
    AtPrepare prepare = {};
    AtMaps maps;
    AtExtra ex = {};
};

// The tensor as bulk copies see it, copied first where they cannot or where masked cells have to be zeros.
int32_t at_operand(const AttnProblem& p, const AttnTensor& t, int heads, int cells, const uint8_t* zeros, bf16* copy,
                   int box_channels, AtHost* h, CUtensorMap* map)
{
    const void* at = t.p;
    long long sc = t.sc, sn = t.sn;
    const bool fits = reinterpret_cast<uintptr_t>(at) % 16 == 0 && sc % 8 == 0 && (p.n == 1 || sn % 8 == 0) && sc > 0
                      && (p.n == 1 || sn > 0);
    if (!fits || zeros)
    {
        const int channels = heads * p.d;
        const long long pitch = (cells + 7) / 8 * 8;
        h->prepare.job[h->prepare.jobs++] = AtCopy{static_cast<const bf16*>(at), copy, sn, sc, zeros, channels, cells,
                                                   (long long) p.n * channels * (pitch / 8)};
        at = copy;
        sc = pitch;
        sn = pitch * channels;
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
    h->ex.status = attn_tc_status();
    DCB_REQUIRE(h->ex.status, "no status word on this device");
    if (p.kv_mask)
    {
        a.mask = p.kv_mask;
        a.bits = p.bits;
        a.cells = p.sk;
        a.words = 4ll * attn_tiles(p.sk, AT_TILE);
        a.words_total = a.words * p.n;
        h->ex.kv_bits = p.bits;
        h->ex.words = a.words;
    }
    const int rows = a.jobs + (p.kv_mask ? 1 : 0);
    if (rows == 0)
        return DCB_OK;
    long long units = a.words_total;
    for (int i = 0; i < a.jobs; ++i)
        units = std::max(units, a.job[i].units);
    const unsigned blocks = (unsigned) std::min<long long>((units + 255) / 256, 16ll * num_sms());
    DCB_CUDA_TRY(launch_overlapped(attn_prepare_kernel, dim3(blocks, rows), 256, 0, stream, a));
    return DCB_OK;
}

} // namespace

// Looked up once per device: a kernel argument must not cost a symbol lookup a call, nor one inside a capture.
int* attn_tc_status()
{
    static thread_local int known_device = -1;
    static thread_local int* known = nullptr;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess)
        return nullptr;
    if (device != known_device)
    {
        void* p = nullptr;
        if (cudaGetSymbolAddress(&p, at_status_word) != cudaSuccess)
        {
            (void) cudaGetLastError();
            return nullptr;
        }
        known = static_cast<int*>(p);
        known_device = device;
    }
    return known;
}

bool attn_tc_apart(const AttnProblem& p)
{
    return p.sq <= AT_TILE && attn_tiles(p.sk, AT_TILE) >= 4;
}

void attn_tc_splits(AttnProblem* p, bool backward)
{
    const long long slots = (p->d <= 64 ? 2 : 1) * num_sms(); // blocks at a time
    const long long q_tiles = attn_tiles(p->sq, AT_TILE), k_tiles = attn_tiles(p->sk, AT_TILE);
    const long long qh = (long long) p->n * p->q_heads, kh = (long long) p->n * p->kv_heads;
    p->q_splits = backward ? attn_splits(kh * k_tiles, (int) std::min<long long>(q_tiles * p->group, 1 << 30), slots, 2)
                           : 1;
    if (!backward && attn_tc_apart(*p))
        p->kv_splits = 2 * attn_splits(qh, (int) k_tiles / 2, num_sms(), 2);
    else
        p->kv_splits = attn_splits(qh * (backward ? q_tiles : (q_tiles + 1) / 2), (int) k_tiles, slots, 2);
}

int32_t attn_tc_fwd(const AttnProblem& p, cudaStream_t stream)
{
    AtHost h;
    const int box = p.d <= 64 ? 64 : 128;
    // masked keys have weight 0, but 0 times what they hold has to be 0: their values are copied as zeros
    if (int32_t e = at_operand(p, p.q, p.q_heads, p.sq, nullptr, p.copy_q, box, &h, &h.maps.q))
        return e;
    if (int32_t e = at_operand(p, p.k, p.kv_heads, p.sk, nullptr, p.copy_k, box, &h, &h.maps.k))
        return e;
    if (int32_t e = at_operand(p, p.v, p.kv_heads, p.sk, p.kv_mask, p.copy_v, box, &h, &h.maps.v))
        return e;
    h.maps.d_o = h.maps.q;
    if (int32_t e = at_prepare(p, &h, stream))
        return e;
    return attn_tc_fwd_launch(p, h.maps, h.ex, stream);
}

int32_t attn_tc_bwd(const AttnProblem& p, cudaStream_t stream)
{
    AtHost h;
    const int box = p.d <= 64 ? 64 : 128;
    // whatever a gradient that is 0 is multiplied with has to be finite
    if (int32_t e = at_operand(p, p.q, p.q_heads, p.sq, p.q_mask, p.copy_q, box, &h, &h.maps.q))
        return e;
    if (int32_t e = at_operand(p, p.k, p.kv_heads, p.sk, p.kv_mask, p.copy_k, box, &h, &h.maps.k))
        return e;
    if (int32_t e = at_operand(p, p.v, p.kv_heads, p.sk, nullptr, p.copy_v, box, &h, &h.maps.v))
        return e;
    if (int32_t e = at_operand(p, p.d_o, p.q_heads, p.sq, p.q_mask, p.copy_do, box, &h, &h.maps.d_o))
        return e;
    if (int32_t e = at_prepare(p, &h, stream))
        return e;
    return attn_tc_bwd_launch(p, h.maps, h.ex, stream);
}

} // namespace dcb
