// Attention on the tensor cores: what its three kernels share.
//
// A tile is 128 cells of one head, [channel][cell] as memory has it, in two halves of 64 cells: a
// half is D rows of 128 bytes, fetched by one bulk tensor copy with the 128-byte swizzle.  The same
// tile serves a product over the channels (cells are the rows or columns: the operand lies
// "across", the reduction index strides over the 128-byte rows) and a product over the cells
// (channels are the columns, the reduction index runs along the rows), so nothing is transposed.
// Scores and their gradients never leave tensor memory but for the registers of the threads that
// own a row; as operand of the second product they go back there, two bf16 to a column, over the
// fp32 values that they were made from.
#pragma once

#include "attention.cuh"
#include "conv_tc_common.cuh"

namespace dcb
{

constexpr int AT_TILE = 128;
// Two teams of 128 for the rows; a warp that issues products, one that issues copies, two that fill up the third
// warpgroup.  384 threads are launched with 168 registers each; the teams take some of the third group's:
// 2 x 216 + 72 = 3 x 168.
constexpr int AT_THREADS = 384;
constexpr int AT_TEAM_REGS = 216, AT_OTHER_REGS = 72;
static_assert(2 * AT_TEAM_REGS + AT_OTHER_REGS <= 3 * 168, "more registers than the block was launched with");
constexpr int AT_MMA_WARP = 8;
constexpr int AT_TMA_WARP = 9;

// A ring of shared-memory slots: use number i of a ring of n has slot i % n, lap i / n.
struct AtRing
{
    uint32_t slot = 0, lap = 0;
    __device__ __forceinline__ void next(uint32_t n)
    {
        if (++slot == n)
        {
            slot = 0;
            ++lap;
        }
    }
};

// The warp that issues products runs converged, and only the instructions themselves are one lane's: their operands are
// then uniform registers, as they want them.  (With one lane running the whole loop an instruction took 140 clocks to
// issue: 12 of them 1700.)
__device__ __forceinline__ uint32_t at_elect()
{
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}

__device__ __forceinline__ void at_commit(uint64_t* bar, uint32_t elected)
{
    if (elected)
        mma_commit(bar);
}

// Both operands in shared memory.
__device__ __forceinline__ void at_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t elected)
{
    asm volatile("{\n\t"
                 ".reg .pred p, e;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 e, %5, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
                 "}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected));
}

// A in tensor memory.
__device__ __forceinline__ void at_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate,
                                          uint32_t elected)
{
    asm volatile("{\n\t"
                 ".reg .pred p, e;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "setp.ne.b32 e, %5, 0;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
                 "}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(elected));
}

// bf16 x bf16 -> fp32, M = 128.  across: cells are that operand's rows, channels the reduction.
__device__ __forceinline__ uint32_t at_idesc(uint32_t n, bool a_across, bool b_across)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) a_across << 15) | ((uint32_t) b_across << 16)
           | (n >> 3 << 17) | ((128u >> 4) << 24);
}

template <int D>
struct AtTile
{
    static constexpr uint32_t HALF = D * 128;    // bytes of 64 cells
    static constexpr uint32_t BYTES = 2 * HALF;
    // The tile as operand across: cells in groups of 64, HALF apart; channels in groups of 8 rows, 1024 bytes apart.
    static __device__ __forceinline__ uint64_t across(uint32_t saddr) { return make_desc(saddr, HALF, 1024, 2); }
    // ... and along: channels in groups of 8 rows, 1024 bytes apart; 16 cells are 32 bytes of a row.
    static __device__ __forceinline__ uint64_t along(uint32_t saddr) { return make_desc(saddr, 16, 1024, 2); }
    // In units of 16 bytes, what 16 channels add to the start address (16 cells, along: 2).
    static __device__ __forceinline__ uint32_t across_step(int k) { return (uint32_t) k * (2048 >> 4); }
};

// d = A B' over the channels, 16 a step: both tiles across, 128 cells of A, N of B.
template <int D, int N>
__device__ __forceinline__ void at_scores(uint32_t d, uint32_t a, uint32_t b, int ksteps, uint32_t elected)
{
    const uint64_t da = AtTile<D>::across(a), db = AtTile<D>::across(b);
    const uint32_t idesc = at_idesc(N, true, true);
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
        if (k < ksteps)
            at_mma_ss(d, da + AtTile<D>::across_step(k), db + AtTile<D>::across_step(k), idesc, k > 0, elected);
}

// d += W B over 64 cells: W in tensor memory, two to a column; B is half a tile.
template <int D>
__device__ __forceinline__ void at_weigh(uint32_t d, uint32_t w, uint32_t b, uint32_t n, bool first, uint32_t elected)
{
    const uint64_t db = AtTile<D>::along(b);
    const uint32_t idesc = at_idesc(n, false, false);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        at_mma_ts(d, w + k * 8, db + k * 2, idesc, !(first && k == 0), elected);
}

__device__ __forceinline__ void at_tma_half(uint32_t dst, const CUtensorMap* map, int cell, int head, int n,
                                            uint64_t* bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(cell), "r"(0), "r"(head), "r"(n)
                 : "memory");
}

// 128 cells of a head; cells and channels that are not there arrive as zeros (and count as bytes).
template <int D>
__device__ __forceinline__ void at_tma_tile(uint32_t dst, const CUtensorMap* map, int cell, int head, int n,
                                            uint64_t* bar)
{
    at_tma_half(dst, map, cell, head, n, bar);
    at_tma_half(dst + AtTile<D>::HALF, map, cell + 64, head, n, bar);
}

template <int D, int CELLS>
__device__ __forceinline__ void at_tma_cells(uint32_t dst, const CUtensorMap* map, int cell, int head, int n,
                                             uint64_t* bar)
{
    if constexpr (CELLS == 64)
        at_tma_half(dst, map, cell, head, n, bar);
    else
        at_tma_tile<D>(dst, map, cell, head, n, bar);
}

// `bytes` from a 16-byte aligned address.
__device__ __forceinline__ void at_bulk(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void at_tmem_ld32(uint32_t taddr, float* v)
{
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i)
        v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void at_tmem_wait_ld()
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void at_tmem_st32(uint32_t taddr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ void at_tmem_st16(uint32_t taddr, const uint32_t* r)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

__device__ __forceinline__ void at_tmem_wait_st()
{
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ float at_max3(float a, float b, float c)
{
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Two floats to an instruction.
__device__ __forceinline__ uint64_t at_pair(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}

__device__ __forceinline__ void at_unpair(uint64_t v, float& lo, float& hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

__device__ __forceinline__ uint64_t at_fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

__device__ __forceinline__ uint64_t at_add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ uint64_t at_mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float at_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x of two numbers of at most 127 without the unit that has ex2: 2^i p(f), i the nearest whole number (from the low
// bits of x + 1.5 2^23, to which 127 is added: they are the exponent of 2^i), p of degree 4 with the least greatest
// relative error on [-1/2, 1/2] (Remez exchange; 2.7e-6 with its coefficients in 32 bits).  0 below -126.5, NaN for NaN.
__device__ __forceinline__ void at_exp2_pair(uint64_t x, float& lo, float& hi)
{
    float a, b;
    at_unpair(x, a, b);
    asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(a) : "f"(a)); // -127
    asm("max.NaN.f32 %0, %1, 0fC2FE0000;" : "=f"(b) : "f"(b));
    x = at_pair(a, b);
    const float magic = 12582912.f + 127.f;
    const uint64_t i = at_add2(x, at_pair(magic, magic));
    const uint64_t f = at_fma2(at_add2(i, at_pair(-magic, -magic)), at_pair(-1.f, -1.f), x);
    uint64_t y = at_fma2(f, at_pair(9.570102e-3f, 9.570102e-3f), at_pair(5.591786e-2f, 5.591786e-2f));
    y = at_fma2(y, f, at_pair(.24024744f, .24024744f));
    y = at_fma2(y, f, at_pair(.6931218f, .6931218f));
    y = at_fma2(y, f, at_pair(.9999993f, .9999993f));
    at_unpair(i, a, b);
    a = __uint_as_float(__float_as_uint(a) << 23);
    b = __uint_as_float(__float_as_uint(b) << 23);
    at_unpair(at_mul2(y, at_pair(a, b)), lo, hi);
}

// A wait of a whole warp: it goes on, or gives up, as one.
__device__ __forceinline__ bool at_warp_wait(uint64_t* bar, uint32_t parity, volatile int* give_up)
{
    return __all_sync(~0u, mbar_wait_t<0>(bar, parity, give_up));
}

// Which of two barriers (of those that `left` names) completes its phase first; -1: gave up.  Bounded like every wait.
__device__ __forceinline__ int at_first_ready(uint64_t* b0, uint64_t* b1, uint32_t left, uint32_t parity,
                                              volatile int* give_up)
{
    const auto done = [&](uint64_t* bar) {
        uint32_t d;
        asm volatile("{\n\t"
                     ".reg .pred p;\n\t"
                     "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.b32 %0, 1, 0, p;\n\t"
                     "}"
                     : "=r"(d)
                     : "r"(smem_u32(bar)), "r"(parity)
                     : "memory");
        return d;
    };
    if (left != 3) // one of them only: the ordinary wait
        return at_warp_wait(left == 1 ? b0 : b1, parity, give_up) ? (int) (left >> 1) : -1;
    const long long begin = clock64();
#pragma unroll 1
    for (uint32_t it = 0; it < (1u << 24); ++it)
    {
        if (__all_sync(~0u, done(b0)))
            return 0;
        if (__all_sync(~0u, done(b1)))
            return 1;
        if ((it & 255) == 255 && __any_sync(~0u, *give_up || clock64() - begin > 500000000ll))
            break;
    }
    *give_up = 1;
    return -1;
}

// One arrival a warp, after all its lanes' work.
__device__ __forceinline__ void at_warp_arrive(uint64_t* bar, int lane)
{
    tc_fence_before();
    __syncwarp();
    if (lane == 0)
        mbar_arrive(bar);
}

// The columns up to `last` among 32, the w-th word from column 0 on.
__device__ __forceinline__ uint32_t at_up_to(int last, int w)
{
    const int left = last - 32 * w + 1;
    return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
}

// Channels [c_lo, c_hi) of an accumulator's rows to a tensor ([channel][cell], this thread's cell is i, negative: none), or
// as a part in fp32.  nothing: no product was taken; zero: this row's result is 0 whatever it holds.
__device__ __forceinline__ void at_store(const AttnTensor& t, float* part, long long nh, long long n, int head, int d,
                                         int i, int cells, float factor, bool zero, bool nothing, uint32_t taddr,
                                         int c_lo, int c_hi)
{
    bf16* out = static_cast<bf16*>(t.p) + n * t.sn + (long long) head * d * t.sc + i;
    float* to = part + nh * d * (long long) cells + i;
    for (int c0 = c_lo; c0 < min(c_hi, d); c0 += 32)
    {
        float v[32];
        if (!nothing)
        {
            at_tmem_ld32(taddr + c0, v);
            at_tmem_wait_ld();
        }
        if (i < 0)
            continue;
#pragma unroll
        for (int c = 0; c < 32; ++c)
            if (c0 + c < d)
            {
                const float x = nothing || zero ? 0.f : v[c] * factor;
                if (part)
                    to[(long long) (c0 + c) * cells] = x;
                else
                    out[(c0 + c) * t.sc] = __float2bfloat16_rn(x);
            }
    }
}

// Which tile and walk (head and part) a block has.  Causal walks differ in length: all heads' longest ones first; else a
// head's blocks lie together, whose keys then stay in L2.
__device__ __forceinline__ int at_block(bool causal, int tiles, long long walks, long long* walk)
{
    const long long b = blockIdx.x;
    *walk = causal ? b % walks : b / tiles;
    return (int) (causal ? b / walks : b % tiles);
}

struct AtMaps
{
    CUtensorMap q, k, v, d_o;
};

// A kernel gave up on a wait: a word of each source file, so that no launch has to look a symbol up.
static __device__ int at_gave_up;

// Reads and clears this file's word.
inline int32_t at_read_status(bool* gave_up)
{
    int word = 0;
    DCB_CUDA_TRY(cudaMemcpyFromSymbol(&word, at_gave_up, sizeof(int)));
    if (word)
    {
        *gave_up = true;
        word = 0;
        DCB_CUDA_TRY(cudaMemcpyToSymbol(at_gave_up, &word, sizeof(int)));
    }
    return DCB_OK;
}

// The end of every kernel: who gave up says so, waits for what he started, and the tensor memory goes back.
template <uint32_t COLUMNS = TC_TMEM_COLS>
__device__ __forceinline__ void at_finish(bool ok, int warp, int lane, uint32_t tmem)
{
    if (!ok && lane == 0)
        atomicExch(&at_gave_up, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    __syncwarp();
    if (warp == AT_MMA_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLUMNS) : "memory");
}

// The 128-byte swizzle goes by address bits: tiles start on multiples of 1024 bytes.
__device__ __forceinline__ bool at_misplaced(uint32_t base)
{
    if ((base & 1023u) == 0)
        return false;
    if (threadIdx.x == 0)
        atomicExch(&at_gave_up, 1);
    return true;
}

template <uint32_t COLUMNS = TC_TMEM_COLS>
__device__ __forceinline__ void at_tmem_alloc(uint32_t* slot)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                 "r"(COLUMNS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

template <int N>
__device__ __forceinline__ void at_more_registers()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <int N>
__device__ __forceinline__ void at_fewer_registers()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Waits, bounded, for copies into slots that nobody waited for because the block gave up.
__device__ __forceinline__ void at_drain(uint64_t* full, uint32_t slots, const AtRing& ring)
{
    int give_up = 0;
    for (uint32_t s = 0; s < slots; ++s)
    {
        // the last lap that slot s was loaded in
        const uint32_t uses = ring.lap + (s < ring.slot);
        if (uses > 0)
            mbar_wait_t<20>(&full[s], (uses - 1) & 1, &give_up);
    }
}

// Few queries against many keys: both teams of a block have the same queries.
bool attn_tc_apart(const AttnProblem& p);
int32_t attn_tc_fwd_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream);
int32_t attn_tc_bwd_launch(const AttnProblem& p, const AtMaps& maps, cudaStream_t stream);
int32_t attn_tc_fwd_status(bool* gave_up);
int32_t attn_tc_bwd_status(bool* gave_up);

} // namespace dcb
