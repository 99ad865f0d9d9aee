// What the parts of attention share: the problem as the kernels see it, the split of a long axis
// and the layout of the workspace.
#pragma once

#include "elem.cuh"

#include <algorithm>

namespace dcb
{

constexpr float ATTN_LOG2E = 1.4426950408889634f;
constexpr int ATTN_MAX_HEAD = 128;

// One tensor: [sample][head][channel of the head][cell], cells contiguous.
struct AttnTensor
{
    void* p;
    long long sn, sc; // element strides of samples and channels
};

// The cells of a side that a mask leaves: the kernels see those only, one after the other.
// Per sample the cells' indices, how many lie before a cell, how many there are.  Null without a mask.
struct AttnSide
{
    int *index, *before, *count; // [n][cells], [n][cells + 1], [n]
};

struct AttnProblem
{
    int n, q_heads, kv_heads, group; // group = query heads of a key head
    int d;                           // channels of a head
    int sq, sk;                      // cells
    int causal, offset;              // j <= i + offset
    float scale;                     // of scores, times log2(e): kernels take powers of two
    AttnTensor q, k, v, o, d_o, dq, dk, dv;
    const uint8_t *q_mask, *kv_mask;
    float* lse;                      // [n][q_heads][sq]
    // Backward: lse in powers of two (+infinity where a cell sees nothing) and sum_d o d_o,
    // [2][n * q_heads][stats_pitch], +infinity and 0 behind the last cell (of q_side, where there is one).
    float* stats;
    long long stats_pitch;
    // Parts of a split axis, joined by a kernel of their own:
    //   forward  [splits][n * q_heads][d][sq] sums and [splits][2][n * q_heads][sq] maxima, sums of weights
    //   backward [splits][n * heads][d][cells] sums
    float *part_o, *part_ml, *part_dq, *part_dk, *part_dv;
    AttnSide q_side, kv_side;
    // Tensor cores: copies of tensors that bulk copies cannot address or whose cells a mask picks, [n][heads * d][pitch]
    // with rows of whole 16 bytes.
    bf16 *copy_q, *copy_k, *copy_v, *copy_do;
    int q_splits, kv_splits; // of the queries' axis (dk, dv), of the keys' axis (o, dq)
};

// One sample's cells on one side, as the kernels count them: all, or those that a mask leaves.
struct AttnCells
{
    int count, cells;
    const int *index, *counted;
    __device__ __forceinline__ AttnCells(const AttnSide& s, long long n, int cells_) : cells(cells_)
    {
        index = s.index ? s.index + n * cells : nullptr;
        counted = s.index ? s.before + n * (cells + 1ll) : nullptr;
        count = s.index ? s.count[n] : cells;
    }
    __device__ __forceinline__ int cell(int r) const { return index ? index[r] : r; }
    // How many lie before cell x of the grid.
    __device__ __forceinline__ int before(long long x) const
    {
        const int c = (int) (x < 0 ? 0 : x > cells ? cells : x);
        return counted ? counted[c] : c;
    }
};

// Row r of the queries sees the first so many keys; later rows see no fewer.
__device__ __forceinline__ int attn_limit(const AttnProblem& p, const AttnCells& q, const AttnCells& kv, int r)
{
    if (r < 0 || r >= q.count)
        return 0;
    return p.causal ? kv.before((long long) q.cell(r) + p.offset + 1) : kv.count;
}

__host__ __device__ inline int attn_tiles(int cells, int tile)
{
    return (cells + tile - 1) / tile;
}

// Splits of a walk over `steps` tiles so that `work` walks fill `slots` blocks; a part walks a tile at least.
inline int attn_splits(long long work, int steps, long long slots)
{
    if (work <= 0 || work >= slots)
        return 1;
    return (int) std::max<long long>(1, std::min<long long>(slots / work, steps));
}

// Kernels of attention_thin.cu: the forward pass of so few queries that it is a pass over the keys.  2 x 8 heads x 64,
// against the other kernels: a bf16 query over 64^2 keys 9 us against 16, over 32^3 36 against 43 (31 x 33 x 31: 72
// against 100), but two queries 52 against 43; eight fp32 queries over 64^2 keys 34 us against 42, over 20 x 20 x 65 227
// against 243.
constexpr int ATTN_THIN_BF16 = 1, ATTN_THIN_F32 = 8; // cells of q
bool attn_thin(const AttnProblem& p, int32_t dtype);
void attn_thin_splits(AttnProblem* p, int32_t dtype);
bool attn_thin_backward(const AttnProblem& p, int32_t dtype);
void attn_thin_bwd_splits(AttnProblem* p);
int32_t attn_thin_bwd(const AttnProblem& p, cudaStream_t stream);
int32_t attn_thin_fwd(const AttnProblem& p, int32_t dtype, cudaStream_t stream);

// Kernels of attention_tc.cu (bf16) and attention_simt.cu (fp32), both behind attn_index, which fills the sides.
int32_t attn_tc_fwd(const AttnProblem& p, cudaStream_t stream);
int32_t attn_tc_bwd(const AttnProblem& p, cudaStream_t stream);
void attn_tc_splits(AttnProblem* p, bool backward);
int32_t attn_tc_status(bool* gave_up); // of the current device, cleared
int32_t attn_simt_fwd(const AttnProblem& p, cudaStream_t stream);
int32_t attn_simt_bwd(const AttnProblem& p, cudaStream_t stream);
void attn_simt_splits(AttnProblem* p, bool backward);

} // namespace dcb
