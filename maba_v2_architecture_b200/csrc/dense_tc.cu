// Products of 16-bit operands on the 5th-generation tensor cores (tcgen05, TMEM, TMA).
//
// The tensor cores truncate when they add to their float32 accumulator, once per 16
// contraction indices: a sum over K loses about K 1e-9 of itself toward zero (measured
// 6e-7 relative at K = 640, 4.4e-6 at 4,096).  That is far below a 16-bit result's rounding,
// but not below a float32 result's, so sums that end in float32 (MODE 1) leave TMEM every
// 640 indices and are added, rounded to nearest, in the epilogue's registers.
//
// Persistent, one CTA per SM.  A work unit is a tile of C (128 rows of A by bn rows of B;
// with CG = 2 a cluster's two CTAs share a tile of 256 rows: each loads its own 128 rows of
// A and one half of B, so a k-block costs an SM 32 KB for 128 x 256 x 64 products instead
// of 48 KB, below what L2 delivers per SM; with this step the gated block of 65,536 x 640 -> 2 x
// 1248 went from 199 to 165 us in a row of calls) over one split of the contraction.  The warps:
//  * epilogue (16, or 8 where they hold a unit's sums): warp w reads TMEM lanes 32 (w & 3)..
//           and every fourth (second) 32-column chunk and applies the epilogue;
//  * TMA producer: 64 contraction indices per stage, 128-byte swizzle, operands K-major or
//           (for the transposed products of the backward pass) MN-major;
//  * MMA:   allocates TMEM and issues the products, one thread (a warp-wide loop with an
//           election for each took 560 cycles to issue a k-block of 512);
//  * side:  brings the epilogue's residual or gradient, 128 rows x 32 columns a copy.
// The float32 accumulator is double-buffered in TMEM (2 x 256 columns): a unit's epilogue
// runs under the next unit's products.  The gated block's tile holds bn/2 rows of w_gate and
// bn/2 of w_up, so a thread sees both projections of an element in its own row.
//
// What bounds it (bf16; one launch, counters and time of a capture): the gated block of 65,536 x
// 640 -> 2 x 1248 takes 137 us, the tensor pipe active 92 % of it; in a row of calls the power limit
// holds the clock near 1.2 GHz and a call takes 174 us.  The linear map with a scale and a float32
// residual, 65,536 x 1248 -> 640, takes 108 us (140 in a row, for the same reason): tensor pipe 57 %,
// DRAM 52 % of its peak, so neither, but the epilogue's chain of TMEM, copy and barrier latencies.
// The gradient pass of a map with a bias, SiLU and scale, 16,384 x 640 -> 2560 with column sums,
// takes 82 us: an instruction issued in 57 % of the cycles, the ALU 47 % busy, the tensor pipe 36 %.
//
// Every mbarrier wait is bounded; a wait that runs out raises the CTA's abort flag, all
// roles leave their loops, copies and products in flight are drained (bounded), TMEM is
// freed and the error word behind maba_device_error() is set.
#include "dense.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

#include <atomic>
#include <cmath>
#include <type_traits>

namespace maba {
namespace dense {

__device__ int g_dense_error = 0;

namespace {
using namespace tc;

// Epilogue warps: 16 where a chunk's registers allow four warps per scheduler (their chains of
// shared-memory, copy and SFU latencies hide each other), 8 where a warp holds a unit's sums.
// Then one warpgroup: TMA of the operands, MMA, TMA of the epilogue's matrix, one idle warp; it
// lends registers to the epilogue's.  What the split hands out is what the block is launched with.
template <int MODE> struct Warps {
    static constexpr int EPI = MODE == 0 ? 16 : 8, TMA = EPI, MMA = EPI + 1, SIDE = EPI + 2, THREADS = (EPI + 4) * 32;
    static constexpr int REG_LAUNCH = MODE == 0 ? 96 : 168, REG_EPI = MODE == 0 ? 104 : 224, REG_OTHER = MODE == 0 ? 64 : 56;
    static constexpr int GROUPS = EPI / 4;     // of four warps that share a chunk's columns
    static constexpr int CHUNKS = 8 / GROUPS;  // a warp's chunks, GROUPS apart, at most
    static constexpr uint32_t VEC_BYTES = 2 * CHUNKS * 32 * 4;  // a warp's scale and bias
    static_assert(EPI * 32 * REG_EPI + 128 * REG_OTHER <= THREADS * REG_LAUNCH, "register split exceeds the launch");
};
constexpr int BK = 64;
constexpr uint32_t A_BYTES = 128 * BK * 2;
constexpr int MAX_STAGES = 8;
constexpr uint32_t BAR_BYTES = 512;
constexpr uint32_t SMEM_MAX = 227 * 1024;
constexpr int TMEM_COLS = 512, ACC_COLS = 256;

enum { B_FULL = 0, B_EMPTY = MAX_STAGES, B_TFULL = 2 * MAX_STAGES, B_TEMPTY = B_TFULL + 2, B_DRAIN = B_TEMPTY + 2,
       B_SFULL = B_DRAIN + 1, B_SEMPTY = B_SFULL + 8, N_BARS = B_SEMPTY + 8 };  // [group][slot]
static_assert(N_BARS * 8 + 8 <= BAR_BYTES, "barrier area");

struct TcArgs {
    int64_t M, N;
    int kblocks, kseg, kb_split;  // contraction blocks over all segments, of one segment, of one split
    int tiles_n, splits, pairs, units;
    int d_inner, d_col, d_row;  // from a worker's unit to its next
    int bn, b_rows;  // columns of the MMA, rows of B per CTA
    int flush;       // contraction blocks between two readings of the accumulator
    int stages;
    uint32_t stage_bytes, load_bytes;  // of shared memory, and of the copies (of both CTAs)
    uint32_t idesc;
    int out_tma;                         // the results leave by copies
    int in_place;                        // from the buffer that brought the residual or gradient
    int n_in, n_out;                     // staging buffers per warp
    uint32_t in_bytes, out_bytes, vec_at, bar_at;  // of one buffer; places of the vectors and the barriers
    Epilogue e;
    float* partial;
    int64_t ldp;
};

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Pairs of float32 in one instruction each: the epilogue's issue slots are what the products
// leave it.
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
// a = a * b + c
__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ float exp2_sfu(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_sfu(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / (1 + e^-z): the SFU's exponential and reciprocal.  The exponential's argument is rounded twice,
// so the result is off by up to (4 + |z|) 2^-23 of itself; below z = -87, where it leaves float32's
// normal range, it is 0
__device__ __forceinline__ void sigmoid2(float z0, float z1, float& s0, float& s1) {
    s0 = z0, s1 = z1;
    mul2(s0, s1, -1.4426950408889634f, -1.4426950408889634f);
    s0 = exp2_sfu(s0), s1 = exp2_sfu(s1);
    add2(s0, s1, 1.f, 1.f);
    s0 = rcp_sfu(s0), s1 = rcp_sfu(s1);
}
// phi and phi' of a pair.
template <int ACT> __device__ __forceinline__ void act2(float& z0, float& z1) {
    if (ACT == ACT_SILU) {
        float s0, s1;
        sigmoid2(z0, z1, s0, s1);
        mul2(z0, z1, s0, s1);
    } else {
        z0 = act_f(z0, ACT), z1 = act_f(z1, ACT);
    }
}
template <int ACT>
__device__ __forceinline__ void act_grad2(float z0, float z1, float& y0, float& y1, float& d0, float& d1) {
    if (ACT == ACT_SILU) {
        float s0, s1;
        sigmoid2(z0, z1, s0, s1);
        y0 = z0, y1 = z1;
        mul2(y0, y1, s0, s1);
        d0 = s0, d1 = s1;  // phi' = s + y (1 - s)
        fma2(d0, d1, -1.f, -1.f, 1.f, 1.f);
        fma2(d0, d1, y0, y1, s0, s1);
    } else {
        act_grad_f(z0, ACT, y0, d0), act_grad_f(z1, ACT, y1, d1);
    }
}
template <typename F> __device__ __forceinline__ void with_act(int act, F f) {
    if (act == ACT_SILU) f(std::integral_constant<int, ACT_SILU>());
    else if (act == ACT_GELU) f(std::integral_constant<int, ACT_GELU>());
    else if (act == ACT_RELU) f(std::integral_constant<int, ACT_RELU>());
    else f(std::integral_constant<int, ACT_NONE>());
}

// --------------------------------------------------------------------------
// The epilogue works on chunks of 32 x 32 elements that tensor-memory copies bring into, and
// take out of, a warp's staging buffers (moved by loads and stores they were bound by the
// load/store unit's address stage).  A buffer has the copy's swizzle: rows of 128 bytes
// (float32) or 64 (16 bits), 16-byte piece p of row r at p ^ (r & 7) or p ^ (r / 2 & 3), so
// that a lane can read its row, or eight lanes a column of pieces, without bank conflicts.
// A result that a copy cannot address (rows not on 16-byte boundaries) is stored element by
// element, out of line; what is read has been made readable.
// --------------------------------------------------------------------------
__device__ __forceinline__ uint4* at32(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint4* at16(unsigned char* st, int row, int piece) {
    return reinterpret_cast<uint4*>(st + row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
}
template <typename E> __device__ __forceinline__ E* element(unsigned char* st, int r, int c) {
    return sizeof(E) == 4 ? reinterpret_cast<E*>(at32(st, r, c >> 2)) + (c & 3)
                          : reinterpret_cast<E*>(at16(st, r, c >> 3)) + (c & 7);
}
// (dst: the chunk's first element)
template <typename E>
__device__ __noinline__ void stage_out(unsigned char* st, E* dst, int64_t ld, int rows, int cols, int lane) {
#pragma unroll 8
    for (int r = 0; r < rows; ++r)
        if (lane < cols) dst[r * ld + lane] = *element<E>(st, r, lane);
}

// A lane's 32 elements of a chunk: its row, or (FRAG, tmem_ld_frag32) the fragment order
// j = 16 b + 4 g + 2 i + e: row 16 b + 8 i + lane / 4, column 8 g + 2 (lane % 4) + e, in which
// a column's 32 rows lie in 8 lanes and its sum takes 7 exchanges for 8 columns, not 31 for 32.
__device__ __forceinline__ int frag_row(int j, int lane) { return (j >> 4) * 16 + ((j >> 1) & 1) * 8 + (lane >> 2); }
__device__ __forceinline__ int frag_col(int j, int lane) { return ((j >> 2) & 3) * 8 + (lane & 3) * 2 + (j & 1); }

// f(j, value, next value) for the 32 elements of a staged chunk, in pairs
template <typename T, bool FRAG, typename F>
__device__ __forceinline__ void with_chunk(bool f32, unsigned char* st, int lane, F f) {
    if (f32) {
        if (FRAG) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float2 x = *reinterpret_cast<const float2*>(element<float>(st, frag_row(j, lane), frag_col(j, lane)));
                f(j, x.x, x.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(at32(st, lane, i));
                f(4 * i, x.x, x.y), f(4 * i + 2, x.z, x.w);
            }
        }
    } else {
        if (FRAG) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float2 x =
                    unpack2<T>(*reinterpret_cast<const uint32_t*>(element<uint16_t>(st, frag_row(j, lane), frag_col(j, lane))));
                f(j, x.x, x.y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = *at16(st, lane, i);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 x = unpack2<T>(w[e]);
                    f(8 * i + 2 * e, x.x, x.y);
                }
            }
        }
    }
}
template <typename T, bool FRAG> __device__ __forceinline__ void put_chunk(const float* z, bool f32, unsigned char* st, int lane) {
    if (f32) {
        if (FRAG) {
#pragma unroll
            for (int j = 0; j < 32; j += 2)
                *reinterpret_cast<float2*>(element<float>(st, frag_row(j, lane), frag_col(j, lane))) = make_float2(z[j], z[j + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(at32(st, lane, i)) = make_float4(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3]);
        }
    } else {
        if (FRAG) {
#pragma unroll
            for (int j = 0; j < 32; j += 2)
                *reinterpret_cast<uint32_t*>(element<uint16_t>(st, frag_row(j, lane), frag_col(j, lane))) = pack2<T>(z[j], z[j + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *at16(st, lane, i) = make_uint4(pack2<T>(z[8 * i], z[8 * i + 1]), pack2<T>(z[8 * i + 2], z[8 * i + 3]),
                                                pack2<T>(z[8 * i + 4], z[8 * i + 5]), pack2<T>(z[8 * i + 6], z[8 * i + 7]));
        }
    }
}
// f(z[j], z[j + 1], v of their columns) for a vector of the chunk's 32 columns in shared memory
template <bool FRAG, typename F> __device__ __forceinline__ void with_vector(float* z, const float* v, int lane, F f) {
    if (FRAG) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float2 x = *reinterpret_cast<const float2*>(v + g * 8 + (lane & 3) * 2);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = (r >> 1) * 16 + g * 4 + (r & 1) * 2;
                f(z[j], z[j + 1], x.x, x.y);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const float4 x = *reinterpret_cast<const float4*>(v + j);
            f(z[j], z[j + 1], x.x, x.y), f(z[j + 2], z[j + 3], x.z, x.w);
        }
    }
}
// Column sums of a chunk (FRAG) over its 32 rows, in a fixed order: v holds a lane's own of its
// eight columns (8 g + 2 (lane % 4) + e at 2 g + e); those of the eight lanes of a column are
// added.  Lane l returns column frag_sum_col(l).
__device__ __forceinline__ int frag_sum_col(int lane) {
    const int q = ((lane >> 4) & 1) * 4 + ((lane >> 3) & 1) * 2 + ((lane >> 2) & 1);
    return (q >> 1) * 8 + (lane & 3) * 2 + (q & 1);
}
__device__ __forceinline__ float frag_column_sum(float* v, int lane) {
#pragma unroll
    for (int o = 16, n = 4; o > 2; o >>= 1, n >>= 1) {
        const bool hi = (lane & o) != 0;
#pragma unroll
        for (int q = 0; q < n; ++q) {
            const float keep = hi ? v[q + n] : v[q], give = hi ? v[q] : v[q + n];
            v[q] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    return v[0];
}

template <typename T, int CG, bool A_MN, bool B_MN, int KIND, int MODE>
__global__ void __launch_bounds__(Warps<MODE>::THREADS, 1)
    tc_kernel(const TcArgs a, const __grid_constant__ CUtensorMap ta0, const __grid_constant__ CUtensorMap ta1,
              const __grid_constant__ CUtensorMap tb0, const __grid_constant__ CUtensorMap tb1,
              const __grid_constant__ CUtensorMap tside, const __grid_constant__ CUtensorMap tout,
              const __grid_constant__ CUtensorMap tout2) {
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* base =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    unsigned char* staging = base + a.stages * a.stage_bytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + a.bar_at);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
    volatile int* abort_f = reinterpret_cast<volatile int*>(tmem_slot + 1);

    constexpr int EPI_WARPS = Warps<MODE>::EPI, W_TMA = Warps<MODE>::TMA, W_MMA = Warps<MODE>::MMA;
    constexpr int W_SIDE = Warps<MODE>::SIDE, GROUPS = Warps<MODE>::GROUPS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
    const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

    if (tid == 0) {
        for (int i = 0; i < N_BARS; ++i)
            mbar_init(&bars[i], i == B_TEMPTY || i == B_TEMPTY + 1 ? EPI_WARPS * CG : (i >= B_SEMPTY ? 4 : 1));
        *abort_f = 0;
        fence_barrier_init();
    }
    if (warp == W_TMA && lane == 0) {
        prefetch_tmap(&ta0);
        prefetch_tmap(&tb0);
    }
    if (warp == W_MMA) {
        if (CG == 2) tmem_alloc_pair<TMEM_COLS>(tmem_slot);
        else tmem_alloc<TMEM_COLS>(tmem_slot);
    }
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // A unit: splits innermost, then the pair index, then columns, then rows of tiles.  A worker
    // walks its units by adding (a division for each took the epilogue longer than a chunk).
    constexpr bool INNER = KIND == E_STORE;  // the others have neither splits nor pairs
    struct Unit {
        int u, inner, col, row;  // index and its digits
        __device__ int pair(const TcArgs& a) const { return INNER && inner >= a.splits ? 1 : 0; }
        __device__ int split(const TcArgs& a) const { return INNER ? inner - pair(a) * a.splits : 0; }
        __device__ int kb0(const TcArgs& a) const { return INNER ? split(a) * a.kb_split : 0; }
        __device__ int kb1(const TcArgs& a) const {
            const int k = INNER ? kb0(a) + a.kb_split : a.kblocks;
            return k < a.kblocks ? k : a.kblocks;
        }
        __device__ int n0(const TcArgs& a) const { return col * (KIND == E_GLU || KIND == E_GLU_BWD ? a.bn / 2 : a.bn); }
    };
    auto row_of = [&](const Unit& t) { return t.row * (128 * CG) + (int)rank * 128; };
    auto first_unit = [&]() {
        Unit t;
        t.u = worker;
        const int inner = INNER ? a.splits * a.pairs : 1, tile = worker / inner;
        t.inner = worker - tile * inner;
        t.row = tile / a.tiles_n, t.col = tile - t.row * a.tiles_n;
        return t;
    };
    auto next_unit = [&](Unit& t) {
        t.u += workers, t.col += a.d_col, t.row += a.d_row;
        if (INNER) {
            t.inner += a.d_inner;
            if (t.inner >= a.splits * a.pairs) t.inner -= a.splits * a.pairs, ++t.col;
        }
        if (t.col >= a.tiles_n) t.col -= a.tiles_n, ++t.row;
    };

    if (warp >= EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Warps<MODE>::REG_OTHER));
    if (warp == W_TMA) {
        // ============================ TMA producer ============================
        // One thread runs the loop: a warp-wide one with an election for each copy took longer
        // to issue a k-block than the tensor cores to multiply it.
        if (elect_one()) {
        int st = 0, it = 0;
        uint32_t phase = 1;  // (a fresh barrier's previous phase counts as complete)
        bool ok = true;
        for (Unit t = first_unit(); t.u < a.units && ok; next_unit(t)) {
            const int m0 = row_of(t), n0 = t.n0(a), kb1 = t.kb1(a), pair = t.pair(a);
            for (int kb = t.kb0(a); kb < kb1; ++kb, ++it) {
                ok = mbar_wait(&bars[B_EMPTY + st], phase, abort_f);
                if (!ok) break;
                const int seg = kb >= a.kseg ? 1 : 0, k0 = (kb - seg * a.kseg) * BK;
                const CUtensorMap* ma = (a.pairs == 2 ? pair : seg) ? &ta1 : &ta0;
                unsigned char* sa = base + st * a.stage_bytes;
                {
                    uint64_t* full = &bars[B_FULL + st];
                    const uint32_t full0 = CG == 2 ? cluster_addr(full, 0) : 0u;
                    auto load = [&](unsigned char* dst, const CUtensorMap* m, int x, int y) {
                        if (CG == 2) tma_load_3d_pair(dst, m, full0, x, y, 0);
                        else tma_load_3d(dst, m, full, x, y, 0);
                    };
                    if (rank == 0) mbar_arrive_expect_tx(full, a.load_bytes);
                    {
                        unsigned char* sb = sa + A_BYTES;
                        if (A_MN) {
                            load(sa, ma, m0, k0);
                            load(sa + A_BYTES / 2, ma, m0 + 64, k0);
                        } else {
                            load(sa, ma, k0, m0);
                        }
                        if (KIND == E_GLU || KIND == E_GLU_BWD) {
                            if (CG == 2) {
                                load(sb, rank ? &tb1 : &tb0, k0, n0);
                            } else {
                                load(sb, &tb0, k0, n0);
                                load(sb + a.bn / 2 * 128, &tb1, k0, n0);
                            }
                        } else {
                            const CUtensorMap* mb = (a.pairs == 2 ? pair : seg) ? &tb1 : &tb0;
                            const int y = n0 + (int)rank * a.b_rows;
                            if (B_MN) {
                                for (int i = 0; i < a.b_rows; i += 64) load(sb + i * 128, mb, y + i, k0);
                            } else {
                                load(sb, mb, k0, y);
                            }
                        }
                    }
                }
                if (++st == a.stages) st = 0, phase ^= 1;
            }
        }
        // every copy has landed (rank 0's barriers count the pair's), and every arrival that rank
        // 0's products make on this CTA's barriers, before it may exit
        for (int s = 0; s < a.stages && s < it; ++s) {
            const uint32_t last = ((it - 1 - s) / a.stages) & 1;
            if (rank == 0) mbar_wait(&bars[B_FULL + s], last, nullptr);
            if (ok) ok = mbar_wait(&bars[B_EMPTY + s], last, abort_f);
        }
        }
    } else if (warp == W_MMA) {
        // ============================ MMA issuer ==============================
        if (rank == 0 && elect_one()) {
            const uint64_t ad0 = sdesc_sw128(smem_addr(base), A_MN ? A_BYTES / 2 : 16, 1024);
            const uint64_t bd0 = sdesc_sw128(smem_addr(base + A_BYTES), B_MN ? 8192 : 16, 1024);
            constexpr uint32_t ak = A_MN ? 2048 >> 4 : 32 >> 4, bk = B_MN ? 2048 >> 4 : 32 >> 4;
            auto mma = [&](uint32_t d, uint64_t ad, uint64_t bd, uint32_t acc) {
                if (CG == 2) umma_f16_ss_pair(d, ad, bd, a.idesc, acc);
                else umma_f16_ss(d, ad, bd, a.idesc, acc);
            };
            auto commit = [&](uint64_t* bar) {
                if (CG == 2) umma_commit_pair(bar);
                else umma_commit(bar);
            };
            int st = 0, buf = 0;
            uint32_t phase = 0, tphase = 1;
            bool ok = true;
            for (Unit t = first_unit(); t.u < a.units && ok; next_unit(t)) {
                const int kb1 = t.kb1(a);
                for (int f0 = t.kb0(a); f0 < kb1; f0 += a.flush) {
                    const int f1 = f0 + a.flush < kb1 ? f0 + a.flush : kb1;
                    const uint32_t d = tmem + buf * ACC_COLS;
                    ok = mbar_wait(&bars[B_TEMPTY + buf], tphase, abort_f);
                    if (!ok) break;
                    tc_fence_after();
                    for (int kb = f0; kb < f1; ++kb) {
                        ok = mbar_wait(&bars[B_FULL + st], phase, abort_f);
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t so = (uint64_t)(st * (a.stage_bytes >> 4));
                        const uint64_t ad = ad0 + so, bd = bd0 + so;
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            const uint32_t acc = kb > f0 || k > 0 ? 1u : 0u;
                            mma(d, ad + k * ak, bd + k * bk, acc);
                        }
                        commit(&bars[B_EMPTY + st]);
                        if (++st == a.stages) st = 0, phase ^= 1;
                    }
                    if (!ok) break;
                    commit(&bars[B_TFULL + buf]);
                    buf ^= 1;
                    if (buf == 0) tphase ^= 1;
                }
            }
            // every product has completed before TMEM is freed
            commit(&bars[B_DRAIN]);
            mbar_wait(&bars[B_DRAIN], 0, nullptr);
            // and the epilogue's last arrivals, of both CTAs, have come in (buffers never used pass)
            for (int i = 0; i < 2 && ok; ++i) {
                ok = mbar_wait(&bars[B_TEMPTY + buf], tphase, abort_f);
                buf ^= 1;
                if (buf == 0) tphase ^= 1;
            }
        }
    } else if (warp == W_SIDE && KIND != E_STORE && KIND != E_GLU) {
        // ================= residual or gradient, chunk by chunk ================
        // One copy brings 32 columns of the CTA's 128 rows, a chunk of each of a group's warps.
        if (a.e.res.p != nullptr && elect_one()) {
            const int width = KIND == E_GLU_BWD ? a.bn / 2 : a.bn;
            uint32_t count[GROUPS] = {};
            bool ok = true;
            for (Unit t = first_unit(); t.u < a.units && ok; next_unit(t)) {
                for (int c0 = 0; c0 * 32 < width && ok; c0 += GROUPS) {
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        const int col = t.n0(a) + (c0 + g) * 32;
                        if (!ok || (c0 + g) * 32 >= width || col >= a.N) continue;
                        const uint32_t n = count[g]++, slot = a.n_in == 2 ? n & 1 : 0, use = a.n_in == 2 ? n >> 1 : n;
                        ok = mbar_wait(&bars[B_SEMPTY + 2 * g + slot], (use & 1) ^ 1, abort_f);
                        if (!ok) continue;
                        uint64_t* full = &bars[B_SFULL + 2 * g + slot];
                        mbar_arrive_expect_tx(full, 4 * a.in_bytes);
                        tma_load_3d(staging + (g * a.n_in + slot) * 4 * a.in_bytes, &tside, full, col, row_of(t), 0);
                    }
                }
            }
            // every copy has landed before the CTA may exit
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
                for (uint32_t back = 1; back <= (uint32_t)a.n_in && back <= count[g]; ++back) {
                    const uint32_t n = count[g] - back, slot = a.n_in == 2 ? n & 1 : 0, use = a.n_in == 2 ? n >> 1 : n;
                    mbar_wait(&bars[B_SFULL + 2 * g + slot], use & 1, nullptr, 200000000ll);
                }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Warps<MODE>::REG_EPI));
        // ============================== epilogue ==============================
        constexpr bool DUAL = KIND == E_GLU || KIND == E_GLU_BWD;
        constexpr bool FRAG = KIND == E_LINEAR_BWD, VECS = KIND == E_LINEAR || KIND == E_LINEAR_BWD;
        constexpr bool SIDE = KIND != E_STORE && KIND != E_GLU;
        constexpr int CH = MODE == 0 ? 1 : 4;  // MODE 1: chunks whose sums a warp holds
        static_assert(MODE == 0 || VECS, "the linear map's kinds alone");
        constexpr int CS = GROUPS, NV = Warps<MODE>::CHUNKS;
        const int q = warp & 3, h = warp >> 2;
        unsigned char* in_buf = staging + (h * a.n_in * 4 + q) * a.in_bytes;  // slots 4 in_bytes apart
        unsigned char* out_buf = staging + EPI_WARPS * a.n_in * a.in_bytes + warp * a.n_out * a.out_bytes;
        float* vscale = reinterpret_cast<float*>(base + a.vec_at + warp * Warps<MODE>::VEC_BYTES);  // [NV chunks][32]
        float* vbias = vscale + NV * 32;
        const Epilogue& e = a.e;
        const int width = DUAL ? a.bn / 2 : a.bn;
        const bool has_side = SIDE && e.res.p != nullptr;
        const bool side_f32 = e.res.f32;
        const bool out_f32 = e.out_f32 || (KIND == E_STORE && a.splits > 1);
        struct Chunk {
            int row0, col0, rows, cols;  // rows, cols: of 32, inside the matrix
        };
        auto place = [&](const Unit& t, int c) {
            Chunk k;
            k.row0 = row_of(t) + q * 32, k.col0 = t.n0(a) + c * 32;
            k.rows = a.M - k.row0 < 32 ? (int)(a.M - k.row0) : 32;
            k.cols = a.N - k.col0 < 32 ? (int)(a.N - k.col0) : 32;
            return k;
        };
        // ---- residual or gradient
        uint32_t used = 0;
        bool ok = true;
        // (in place: a chunk's result is put over what was read and leaves from there, so its
        // buffer goes back to the side warp when the next chunk is asked for, its copy out read)
        int leaving = -1;
        auto side_ready = [&]() {
            if (leaving >= 0) {
                if (lane == 0) {
                    bulk_wait_read<0>();
                    mbar_arrive(&bars[B_SEMPTY + 2 * h + leaving]);
                }
                leaving = -1;
            }
            const uint32_t slot = a.n_in == 2 ? used & 1 : 0, use = a.n_in == 2 ? used >> 1 : used;
            ok = mbar_wait_warp(&bars[B_SFULL + 2 * h + slot], use & 1, abort_f);
            return in_buf + slot * 4 * a.in_bytes;
        };
        auto side_used = [&](bool stays) {
            __syncwarp();
            const int slot = a.n_in == 2 ? (int)(used & 1) : 0;
            if (stays) leaving = slot;
            else if (lane == 0) mbar_arrive(&bars[B_SEMPTY + 2 * h + slot]);
            ++used;
        };
        // ---- results
        uint32_t stored = 0;
        auto store = [&](const Chunk& k, const float* z, const CUtensorMap* map, void* dst, int64_t ld, int plane,
                         unsigned char* in) {
            unsigned char* buf = in;
            if (in == nullptr) {
                buf = out_buf + (a.n_out == 2 ? (stored & 1) * a.out_bytes : 0u);
                ++stored;
                if (lane == 0) {
                    if (a.n_out == 2) bulk_wait_read<1>();
                    else bulk_wait_read<0>();
                }
                __syncwarp();
            }
            put_chunk<T, FRAG>(z, out_f32, buf, lane);
            if (a.out_tma) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_3d(map, buf, k.col0, k.row0, plane);
                    bulk_commit();
                }
            } else {
                __syncwarp();
                if (out_f32) stage_out<float>(buf, static_cast<float*>(dst) + k.row0 * ld + k.col0, ld, k.rows, k.cols, lane);
                else stage_out<uint16_t>(buf, static_cast<uint16_t*>(dst) + k.row0 * ld + k.col0, ld, k.rows, k.cols, lane);
                __syncwarp();
            }
        };
        // ---- scale and bias of a unit's columns, one unit ahead in registers, as they are in
        // memory (a conversion here would wait for each load in turn)
        uint32_t ps[NV], pb[NV];
        auto bits_at = [&](const Side& v, int col) {
            const int64_t i = col * v.sc;
            return v.f32 ? static_cast<const uint32_t*>(v.p)[i] : (uint32_t)static_cast<const uint16_t*>(v.p)[i];
        };
        auto value_of = [&](const Side& v, uint32_t bits) {
            if (!v.f32) return unpack2<T>(bits).x;
            return __uint_as_float(bits);
        };
        auto fetch_vectors = [&](const Unit& t) {
#pragma unroll
            for (int cc = 0; cc < (VECS ? NV : 0); ++cc) {
                const int col = t.n0(a) + (h + CS * cc) * 32 + lane;
                const bool in = (h + CS * cc) * 32 < width && col < a.N;
                ps[cc] = pb[cc] = 0u;  // (columns past the last are not stored)
                if (in && e.scale.p) ps[cc] = bits_at(e.scale, col);
                if (in && e.bias.p) pb[cc] = bits_at(e.bias, col);
            }
        };
        // ---- accumulators
        int buf = 0;
        uint32_t phase = 0;
        auto wait_full = [&]() {
            ok = mbar_wait_warp(&bars[B_TFULL + buf], phase, abort_f);
            tc_fence_after();
            return ok;
        };
        auto release = [&]() {  // this warp has read its part
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(cluster_addr(&bars[B_TEMPTY + buf], 0));
                else mbar_arrive(&bars[B_TEMPTY + buf]);
            }
            __syncwarp();
            buf ^= 1;
            if (buf == 0) phase ^= 1;
        };
        auto load_sums = [&](float* z, uint32_t at) {
            __syncwarp();  // (a warp-wide instruction; one lane may come from issuing a copy)
            if (FRAG) tmem_ld_frag32(at, reinterpret_cast<uint32_t*>(z));
            else tmem_ld32(at, reinterpret_cast<uint32_t*>(z));
        };
        // ---- one chunk
        auto chunk = [&](const Unit& t, int c, float* z, float* w) {
            const Chunk k = place(t, c);
            if (k.cols <= 0) return;
            if (k.rows <= 0) {  // (the group's copy still counts this warp)
                if (has_side) side_ready(), side_used(false);
                return;
            }
            unsigned char* in = nullptr;
            const float *vs = vscale + c / CS * 32, *vb = vbias + c / CS * 32;
            if (KIND == E_LINEAR) {
                if (e.bias.p) with_vector<FRAG>(z, vb, lane, add2);
                with_act(e.act, [&](auto A) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) act2<A.value>(z[j], z[j + 1]);
                });
                if (e.scale.p) with_vector<FRAG>(z, vs, lane, mul2);
                if (has_side) {
                    in = side_ready();
                    with_chunk<T, FRAG>(side_f32, in, lane, [&](int j, float g0, float g1) { add2(z[j], z[j + 1], g0, g1); });
                    side_used(a.in_place);
                }
            } else if (KIND == E_LINEAR_BWD) {
                float sb[8] = {}, ss[8] = {};  // this lane's part of its eight columns' sums
                if (e.bias.p) with_vector<FRAG>(z, vb, lane, add2);
                in = side_ready();
                with_act(e.act, [&](auto A) {
                    with_chunk<T, FRAG>(side_f32, in, lane, [&](int j, float g0, float g1) {
                        float y0, y1, d0, d1;
                        act_grad2<A.value>(z[j], z[j + 1], y0, y1, d0, d1);
                        if (k.rows < 32 && frag_row(j, lane) >= k.rows) y0 = y1 = d0 = d1 = 0.f;  // whatever the bias is
                        const int c = ((j >> 2) & 3) * 2;
                        z[j] = g0, z[j + 1] = g1;
                        mul2(z[j], z[j + 1], d0, d1);
                        fma2(y0, y1, g0, g1, ss[c], ss[c + 1]);
                        ss[c] = y0, ss[c + 1] = y1;
                    });
                });
                side_used(a.in_place);
                if (e.scale.p) with_vector<FRAG>(z, vs, lane, mul2);
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    if (k.rows < 32 && frag_row(j, lane) >= k.rows) continue;  // whatever the scale is
                    add2(sb[((j >> 2) & 3) * 2], sb[((j >> 2) & 3) * 2 + 1], z[j], z[j + 1]);
                }
                const int col = frag_sum_col(lane);
                const int64_t at = (int64_t)(k.row0 >> 5) * a.N + k.col0 + col;
                if (e.part_bias) {
                    const float s = frag_column_sum(sb, lane);
                    if (col < k.cols) e.part_bias[at] = s;
                }
                if (e.part_scale) {
                    const float s = frag_column_sum(ss, lane);
                    if (col < k.cols) e.part_scale[at] = s;
                }
            } else if (KIND == E_GLU) {
                with_act(e.act, [&](auto A) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        act2<A.value>(z[j], z[j + 1]);
                        mul2(z[j], z[j + 1], w[j], w[j + 1]);
                    }
                });
            } else if (KIND == E_GLU_BWD) {
                in = side_ready();
                with_act(e.act, [&](auto A) {
                    with_chunk<T, FRAG>(side_f32, in, lane, [&](int j, float g0, float g1) {
                        float y0, y1, d0, d1;
                        act_grad2<A.value>(z[j], z[j + 1], y0, y1, d0, d1);
                        mul2(d0, d1, w[j], w[j + 1]);
                        w[j] = g0, w[j + 1] = g1;
                        z[j] = g0, z[j + 1] = g1;
                        mul2(w[j], w[j + 1], y0, y1);
                        mul2(z[j], z[j + 1], d0, d1);
                    });
                });
                side_used(false);
            }
            if (KIND == E_STORE && a.splits > 1) {
                const int part = t.split(a) * a.pairs + t.pair(a);
                store(k, z, &tout, a.partial + (int64_t)part * a.M * a.ldp, a.ldp, part, nullptr);
            } else {
                const bool second = t.pair(a) != 0;
                store(k, z, second ? &tout2 : &tout, second ? e.out2 : e.out, e.ldo, 0, a.in_place ? in : nullptr);
            }
            if (KIND == E_GLU_BWD) store(k, w, &tout2, e.out2, e.ldo, 0, nullptr);
        };

        Unit t = first_unit();
        if (t.u < a.units) fetch_vectors(t);
        while (t.u < a.units) {
            Unit after = t;
            next_unit(after);
            if (VECS) {
                __syncwarp();
#pragma unroll
                for (int cc = 0; cc < NV; ++cc) {
                    vscale[cc * 32 + lane] = value_of(e.scale, ps[cc]);
                    vbias[cc * 32 + lane] = value_of(e.bias, pb[cc]);
                }
                __syncwarp();
                if (after.u < a.units) fetch_vectors(after);
            }
            if constexpr (MODE != 0) {
                float sz[CH][32], none[1];  // the unit's accumulations, added up
#pragma unroll
                for (int j = 0; j < 32; ++j)
#pragma unroll
                    for (int cc = 0; cc < CH; ++cc) sz[cc][j] = 0.f;
                const int kb1 = t.kb1(a);
                for (int f0 = t.kb0(a); f0 < kb1; f0 += a.flush) {
                    if (!wait_full()) break;
                    const uint32_t acc = tmem + buf * ACC_COLS + ((uint32_t)(q * 32) << 16);
#pragma unroll
                    for (int cc = 0; cc < CH; ++cc) {
                        if ((h + CS * cc) * 32 >= width) continue;
                        float z[32];
                        load_sums(z, acc + (h + CS * cc) * 32);
                        tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
#pragma unroll
                        for (int j = 0; j < 32; ++j) sz[cc][j] += z[j];
                    }
                    release();
                }
                if (!ok) break;
#pragma unroll
                for (int cc = 0; cc < CH; ++cc) {
                    const int c = h + CS * cc;
                    if (c * 32 < width) chunk(t, c, sz[cc], none);
                }
            } else {
                if (!wait_full()) break;
                const uint32_t acc = tmem + buf * ACC_COLS + ((uint32_t)(q * 32) << 16);
                if (h * 32 >= width) release();
                for (int c = h; c * 32 < width; c += CS) {
                    float z[32], w[DUAL ? 32 : 1];
                    load_sums(z, acc + c * 32);
                    if (DUAL) load_sums(w, acc + width + c * 32);
                    tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(z));
                    if (DUAL) tmem_wait_ld_pin32(reinterpret_cast<uint32_t*>(w));
                    if ((c + CS) * 32 >= width) release();
                    chunk(t, c, z, w);
                }
            }
            if (!ok) break;
            t = after;
        }
        if (lane == 0) bulk_wait_all();  // the copies out end before the CTA may
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) {
        // the last arrival that rank 0's products make on this CTA's barriers
        if (rank == 1 && warp == W_MMA) mbar_wait_warp(&bars[B_DRAIN], 0, nullptr);
        cluster_sync();
    }
    if (warp == W_MMA) {
        tc_fence_after();
        if (CG == 2) tmem_dealloc_pair<TMEM_COLS>(tmem);
        else tmem_dealloc<TMEM_COLS>(tmem);
    }
    // the pair frees its TMEM together: neither CTA may be gone, or another in its place, before
    if (CG == 2) cluster_sync();
    if (tid == 0 && *abort_f) atomicExch(&g_dense_error, 1);
}

// --------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------
inline int b_rows_of(int cg, int bn) { return bn / cg; }
inline uint32_t b_bytes_of(int cg, int bn, bool mn) {
    const int r = b_rows_of(cg, bn);
    return (uint32_t)(mn ? (r + 63) / 64 * 64 : r) * 128u;
}

// How a product's sums are kept: 0 one accumulation (16-bit results), 1 added up in registers
// every 640 indices (results, or column sums, that are float32).
int mode_of(const Product& p) {
    if (p.e.kind == E_LINEAR_BWD) return p.e.sums_f32 && p.K > 640 ? 1 : 0;
    return p.e.kind == E_LINEAR && p.e.out_f32 ? 1 : 0;
}

// The tile and the splits with the least estimated time.  Per k-block and SM: the larger of
// the products (128 x bn x 64 at 4,096 per cycle) and the loads (60 bytes per cycle from L2);
// a unit that is not hidden under another adds its fill and epilogue.  The registers that
// hold a unit's sums bound bn in mode 1.  Splits also bound what one accumulation
// truncates: at most 16,384 indices.
Plan plan_of(const Product& p, int mode, double* time) {
    const bool dual = p.form == F_DUAL, store = p.e.kind == E_STORE;
    const int kblocks = (int)ceil_div(p.K, BK) * (p.form == F_SUM ? 2 : 1);
    const int pairs = p.form == F_PAIR ? 2 : 1;
    const int fewest = store && mode == 0 ? (kblocks + 255) / 256 : 1;
    const double out = 8.0 * pairs * (double)p.M * (double)p.N / 3500.0;  // one split's sums, written and read
    Plan best;
    double least = 1e300;
    for (int cg = 1; cg <= 2; ++cg) {
        const int most = cg == 2 ? 256 : 192, slots = sm_count() / cg;
        const int m = (int)((p.M + 128 * cg - 1) / (128 * cg)), n = (int)p.N;
        const double rows = (double)m * pairs;
        for (int bn = dual ? 64 : 32; bn <= most; bn += dual ? 64 : 32) {
            const int cols = dual ? bn / 2 : bn;
            const double tiles = rows * (n / cols + (n % cols != 0));
            const double mma = 2.0 * bn, load = (A_BYTES + b_bytes_of(cg, bn, p.b_mn)) / 60.0;
            const double kcost = mma > load ? mma : load;
            // as few splits as may be, or as many as fill the GPU once, twice (up to 15 more)
            for (int i = 0; i < (store ? 3 : 1); ++i) {
                const double fill = i * (slots / tiles);
                const int ask = i == 0 || fill < fewest ? fewest : (fill > fewest + 15 ? fewest + 15 : (int)fill);
                const int kb = (kblocks + ask - 1) / ask;    // blocks of a split
                const int splits = (kblocks + kb - 1) / kb;  // none of them empty
                const double waves = std::ceil(tiles * splits / slots);
                // (a bit more for the partial sums: a second kernel)
                const double t = waves * kb * kcost + 2000.0 + 12.0 * bn + (splits > 1 ? 2000.0 + splits * out : 0.0);
                if (t < least) least = t, best.cg = cg, best.bn = bn, best.splits = splits;
            }
        }
    }
    *time = least;
    return best;
}

// One operand's map: rows x contraction, read K-major (contraction contiguous) or
// MN-major.
bool operand_map(CUtensorMap* m, int dt, const Matrix& x, int64_t rows, int64_t k, bool mn, int box_rows) {
    const int64_t dims[3] = {mn ? rows : k, mn ? k : rows, 1};
    const int64_t ld = dims[1] > 1 ? (mn ? x.sk : x.sr) : (dims[0] + 7) / 8 * 8;
    const int64_t strides[2] = {ld, ld};
    const uint32_t box[3] = {(uint32_t)BK, (uint32_t)(mn ? BK : box_rows), 1};
    return make_map(m, dt, x.p, 3, dims, strides, box);
}

// The place of a matrix that the epilogue reads or writes in chunks, rows x cols (x parts, one after
// another), in elements of el bytes; false where copies cannot address it.
struct ChunkLayout {
    int64_t dims[3], strides[2];
};
bool chunk_layout(ChunkLayout* c, int el, const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t parts) {
    // one row's stride is never used, whatever the caller's is; parts lie rows * ld apart even so
    if (rows == 1 && parts == 1) ld = (cols + 7) / 8 * 8;
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0 || (ld * el) % 16 != 0 || ld < cols) return false;
    *c = {{cols, rows, parts}, {ld, parts > 1 ? rows * ld : ld}};
    return true;
}
bool chunk_map(CUtensorMap* m, int dt, const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t parts,
               uint32_t box_rows = 32) {
    ChunkLayout c;
    const uint32_t box[3] = {32, box_rows, 1};
    return chunk_layout(&c, dt == MABA_F32 ? 4 : 2, p, rows, cols, ld, parts) && make_map(m, dt, p, 3, c.dims, c.strides, box);
}

using Kernel = void (*)(const TcArgs, const CUtensorMap, const CUtensorMap, const CUtensorMap, const CUtensorMap,
                        const CUtensorMap, const CUtensorMap, const CUtensorMap);

// A kernel ready to launch on the current device: its shared memory limit raised, and the
// device's context bound to this thread, which encoding a tensor map needs (autograd's threads
// come without one).  The register split assumes REG_LAUNCH registers per thread at launch; with
// fewer, the epilogue's increase would never complete, so such a build is refused.
template <typename T, int CG, bool A_MN, bool B_MN, int KIND, int MODE> int ready(Kernel* out, int device) {
    static std::atomic<uint64_t> done{0};
    static thread_local uint64_t bound = 0;
    const auto kern = tc_kernel<T, CG, A_MN, B_MN, KIND, MODE>;
    *out = kern;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if ((done.load(std::memory_order_relaxed) & bound & bit) != 0) return MABA_OK;
    cudaFuncAttributes fa{};
    cudaError_t e = cudaFuncGetAttributes(&fa, kern);
    if (e == cudaSuccess && fa.numRegs != Warps<MODE>::REG_LAUNCH)
        return set_error(MABA_ERR_UNSUPPORTED, "dense(tcgen05): built with %d registers", fa.numRegs);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX);
    if (e != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(e));
    done.fetch_or(bit, std::memory_order_relaxed);
    bound |= bit;
    return MABA_OK;
}

template <typename T, int CG> int kernel_of(Kernel* k, const Product& p, int mode, int device) {
    if (mode == 1)
        return p.e.kind == E_LINEAR ? ready<T, CG, false, false, E_LINEAR, 1>(k, device)
                                    : ready<T, CG, false, false, E_LINEAR_BWD, 1>(k, device);
    switch (p.e.kind) {
        case E_LINEAR: return ready<T, CG, false, false, E_LINEAR, 0>(k, device);
        case E_LINEAR_BWD: return ready<T, CG, false, false, E_LINEAR_BWD, 0>(k, device);
        case E_GLU: return ready<T, CG, false, false, E_GLU, 0>(k, device);
        case E_GLU_BWD: return ready<T, CG, false, false, E_GLU_BWD, 0>(k, device);
        default:
            if (p.a_mn) return ready<T, CG, true, true, E_STORE, 0>(k, device);
            return p.b_mn ? ready<T, CG, false, true, E_STORE, 0>(k, device) : ready<T, CG, false, false, E_STORE, 0>(k, device);
    }
}

}  // namespace

bool tc_readable(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t col_stride) {
    if (col_stride != 1 && cols > 1) return false;
    if ((reinterpret_cast<uintptr_t>(p) & 15u) != 0) return false;
    return rows == 1 || (ld % 8 == 0 && ld >= cols);
}

int64_t partials_reach(int64_t rows, int64_t cols, int64_t ldp, int64_t parts) {
    ChunkLayout c;
    if (!chunk_layout(&c, 4, nullptr, rows, cols, ldp, parts)) return (parts * rows - 1) * ldp + cols;
    return (parts - 1) * c.strides[1] + (rows - 1) * c.strides[0] + cols;
}

Product split_sums(const Product& p) {
    Product q = p;
    q.form = p.form == F_DUAL ? F_PAIR : p.form;
    if (p.form == F_DUAL) q.a[1] = p.a[0];
    q.e = Epilogue{};
    return q;
}

// A product with an epilogue whose few tiles have a long contraction: its sums by splits,
// then the epilogue, where the model says that this is sooner (bf16, whole and split: 100 x 4,000 ->
// 40 16.1 and 11.9 us, -> 640 16.3 and 11.3; the gated block -> 2 x 640 15.7 and 10.9; the gradient
// pass of 24 x 3,776 -> 120 18.4 and 13.6).  A float32 result keeps its bound on one accumulation,
// 640 indices.
Plan tc_plan(const Product& p) {
    const int mode = mode_of(p);
    double whole, split;
    const Plan plan = plan_of(p, mode, &whole);
    if (p.e.kind == E_STORE || p.K < 16 * BK) return plan;
    const int64_t tiles = ceil_div(p.M, 128 * plan.cg) * ceil_div(p.N, p.form == F_DUAL ? plan.bn / 2 : plan.bn);
    if (2 * tiles * plan.cg > sm_count()) return plan;
    Plan parts = plan_of(split_sums(p), mode == 1 ? 0 : mode, &split);
    // (the two more launches cost about 3 us)
    if (parts.splits == 1 || split + 6000.0 >= 0.7 * whole) return plan;
    if (mode == 1 && ceil_div(ceil_div(p.K, BK), parts.splits) > 640 / BK) return plan;
    parts.finish = true;
    return parts;
}

template <typename T>
int tc_product(const Product& p, const Plan& pl, float* partial, int64_t ldp, cudaStream_t s) {
    if (encode_fn() == nullptr) return set_error(MABA_ERR_CUDA, "dense: cuTensorMapEncodeTiled not found");
    constexpr int dt = std::is_same<T, __nv_bfloat16>::value ? MABA_BF16 : MABA_F16;
    const int mode = mode_of(p);
    const bool dual = p.form == F_DUAL, a_mn = p.a_mn, b_mn = p.b_mn;
    TcArgs a{};
    a.M = p.M, a.N = p.N;
    a.kseg = (int)ceil_div(p.K, BK);
    a.kblocks = a.kseg * (p.form == F_SUM ? 2 : 1);
    a.pairs = p.form == F_PAIR ? 2 : 1;
    a.kb_split = (int)ceil_div(a.kblocks, pl.splits);
    a.splits = (int)ceil_div(a.kblocks, a.kb_split);
    a.bn = pl.bn;
    a.b_rows = b_rows_of(pl.cg, pl.bn);
    a.tiles_n = (int)ceil_div(p.N, dual ? pl.bn / 2 : pl.bn);
    const int64_t units = ceil_div(p.M, 128 * pl.cg) * a.tiles_n * a.pairs * a.splits;
    if (units > 0x7fffffff) return set_error(MABA_ERR_UNSUPPORTED, "dense: %lld tiles", (long long)units);
    a.units = (int)units;
    const int slots = sm_count() / pl.cg, workers = a.units < slots ? a.units : slots;
    a.d_inner = workers % (a.splits * a.pairs);
    a.d_col = workers / (a.splits * a.pairs) % a.tiles_n;
    a.d_row = workers / (a.splits * a.pairs) / a.tiles_n;
    const uint32_t bb = b_bytes_of(pl.cg, pl.bn, b_mn);
    a.flush = mode == 0 ? a.kblocks : 640 / BK;
    a.stage_bytes = A_BYTES + (bb + 1023) / 1024 * 1024;
    a.load_bytes = (A_BYTES + bb) * pl.cg;
    // staging: two buffers each way where that leaves enough stages for the products, else fewer
    const int epi = mode == 0 ? Warps<0>::EPI : Warps<1>::EPI, threads = mode == 0 ? Warps<0>::THREADS : Warps<1>::THREADS;
    const bool vecs = p.e.kind == E_LINEAR || p.e.kind == E_LINEAR_BWD;
    const uint32_t vec_bytes = !vecs ? 0 : epi * (mode == 0 ? Warps<0>::VEC_BYTES : Warps<1>::VEC_BYTES);
    const bool out_f32 = p.e.out_f32 || a.splits > 1, side_f32 = p.e.res.f32;
    a.in_bytes = p.e.res.p ? (side_f32 ? 4096 : 2048) : 0;
    a.out_bytes = out_f32 ? 4096 : 2048;
    const uint32_t fixed = 1024 + BAR_BYTES + vec_bytes;
    uint32_t staging = 0;
    a.in_place = p.e.res.p && vecs && side_f32 == out_f32;
    if (a.in_place) a.out_bytes = 0;
    for (int t = 0; t < 3; ++t) {
        a.n_in = t < 2 ? 2 : 1, a.n_out = t < 1 ? 2 : 1;
        staging = epi * (a.n_in * a.in_bytes + a.n_out * a.out_bytes);
        a.stages = (int)((SMEM_MAX - fixed - staging) / a.stage_bytes);
        if (a.stages >= (a.in_place ? 4 : 5)) break;
    }
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    a.vec_at = a.stages * a.stage_bytes + staging;
    a.bar_at = a.vec_at + vec_bytes;
    const size_t smem = 1024 + a.bar_at + BAR_BYTES;
    a.idesc = idesc_f16(128 * pl.cg, pl.bn, dt == MABA_BF16, a_mn, b_mn);
    a.e = p.e;
    a.partial = partial;
    a.ldp = ldp;
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(err));
    Kernel kern = nullptr;
    MABA_TRY((pl.cg == 2 ? kernel_of<T, 2>(&kern, p, mode, device) : kernel_of<T, 1>(&kern, p, mode, device)));
    CUtensorMap m[7];
    const int na = p.form == F_SUM || p.form == F_PAIR ? 2 : 1, nb = na == 2 || dual ? 2 : 1;
    const int box = dual ? pl.bn / 2 : a.b_rows;
    bool ok = true;
    for (int i = 0; i < na; ++i) ok = ok && operand_map(&m[i], dt, p.a[i], p.M, p.K, a_mn, 128);
    for (int i = 0; i < nb; ++i) ok = ok && operand_map(&m[2 + i], dt, p.b[i], p.N, p.K, b_mn, box);
    if (!ok) return set_error(MABA_ERR_CUDA, "dense: tensor map refused");
    if (na == 1) m[1] = m[0];
    if (nb == 1) m[3] = m[2];
    m[4] = m[5] = m[6] = m[0];
    if (p.e.res.p && !chunk_map(&m[4], side_f32 ? MABA_F32 : dt, p.e.res.p, p.M, p.N, p.e.res.sr, 1, 128))
        return set_error(MABA_ERR_CUDA, "dense: tensor map refused");
    if (a.splits > 1) {
        a.out_tma = chunk_map(&m[5], MABA_F32, partial, p.M, p.N, ldp, a.splits * a.pairs);
    } else {
        a.out_tma = chunk_map(&m[5], out_f32 ? MABA_F32 : dt, p.e.out, p.M, p.N, p.e.ldo, 1) &&
                    (!p.e.out2 || chunk_map(&m[6], out_f32 ? MABA_F32 : dt, p.e.out2, p.M, p.N, p.e.ldo, 1));
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(workers * pl.cg));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.cg;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pl.cg == 2 ? 1 : 0;
    err = cudaLaunchKernelEx(&cfg, kern, a, m[0], m[1], m[2], m[3], m[4], m[5], m[6]);
    if (err != cudaSuccess) return set_error(MABA_ERR_CUDA, "dense(tcgen05): %s", cudaGetErrorString(err));
    return check_launch("dense(tcgen05)");
}
template int tc_product<__half>(const Product&, const Plan&, float*, int64_t, cudaStream_t);
template int tc_product<__nv_bfloat16>(const Product&, const Plan&, float*, int64_t, cudaStream_t);

int device_error_take(cudaStream_t s, int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_dense_error, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return set_error(MABA_ERR_CUDA, "device_error: %s", cudaGetErrorString(e));
    const int zero = 0;
    if (v != 0) cudaMemcpyToSymbolAsync(g_dense_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, s);
    *out = v;
    return MABA_OK;
}

}  // namespace dense
}  // namespace maba
